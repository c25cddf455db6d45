"""s2_group_norm against a float64 form: every type and vector width, groups of
one to all channels, one pixel to many chunks, strides, in place, means many
deviations large, and what an infinity or NaN reaches."""
import pytest

from seedvr2_ncnn_amd import capi

pytestmark = pytest.mark.gpu

# (frames, pixels, channels, groups): one value; one pixel; groups of 1, 3, 4, 12, 16
# channels; channel counts that 8, 4 or 1 divide; all channels one group and each its
# own; more channel vectors than threads; several chunks, the last one short
SHAPES = [(1, 1, 1, 1), (2, 1, 512, 32), (1, 64, 512, 32), (3, 77, 33, 11), (1, 1025, 12, 3),
          (2, 300, 60, 5), (1, 5000, 108, 9), (2, 200, 640, 1), (1, 129, 96, 96), (1, 33, 4096, 1),
          (1, 20, 4095, 5), (5, 2049, 128, 32), (1, 40001, 8, 2)]
TYPES = ["float32", "bfloat16", "float16"]


def _draw(shape, dtype, seed, offset=1.0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f, p, c = shape
    x = torch.randn(f, p, c, generator=gen, device="cuda")
    x = x * (0.5 + torch.rand(c, generator=gen, device="cuda"))
    x = x + offset * torch.randn(c, generator=gen, device="cuda")
    gamma = 1 + 0.1 * torch.randn(c, generator=gen, device="cuda")
    beta = 0.1 * torch.randn(c, generator=gen, device="cuda")
    return x.to(getattr(torch, dtype)), gamma, beta


def _check(x, groups, gamma, beta, eps, act, got):
    import row_operators as ro
    want, bound = ro.group_norm(x, groups, gamma, beta, eps, act, got.dtype)
    ro.check(got, want, bound)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_shapes(shape, dtype):
    import torch
    f, p, c, g = shape
    x, gamma, beta = _draw((f, p, c), dtype, p + c)
    got = capi.group_norm(x, g, gamma, beta, 1e-6, capi.ACT_SILU, out_dtype=torch.float32)
    _check(x, g, gamma, beta, 1e-6, "silu", got)


@pytest.mark.parametrize("act", ["none", "gelu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("y_type", TYPES)
def test_types_and_activations(act, x_type, y_type):
    import torch
    import row_operators as ro
    for c, g in ((64, 8), (36, 4), (35, 7)):
        x, gamma, beta = _draw((2, 301, c), x_type, c)
        for gm, bt in ((gamma, beta), (None, None)):
            got = capi.group_norm(x, g, gm, bt, 1e-5, ro.ACTS[act], out_dtype=getattr(torch, y_type))
            _check(x, g, gm, bt, 1e-5, act, got)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_in_place(dtype):
    """Rows inside a wider buffer (pads of 8, 4 and 1 elements), frames interleaved
    by pixel, broadcast frames, and in place; what lies between the rows stays."""
    import torch
    dt = getattr(torch, dtype)
    for c, pad in ((64, 8), (64, 4), (64, 1), (40, 3)):
        x, gamma, beta = _draw((3, 150, c), dtype, pad)
        wide = torch.full((3, 150, c + pad), 7.0, dtype=dt, device="cuda")
        wide[:, :, :c] = x
        out = torch.full((3, 150, c + 2 * pad), -3.0, dtype=dt, device="cuda")
        capi.group_norm(wide[:, :, :c], 8, gamma, beta, out=out[:, :, pad:pad + c])
        _check(x, 8, gamma, beta, 1e-6, "none", out[:, :, pad:pad + c])
        assert (out[:, :, :pad] == -3).all() and (out[:, :, pad + c:] == -3).all()
        inter = x.transpose(0, 1).contiguous().transpose(0, 1)   # [pixels][frames][channels]
        capi.group_norm(inter, 8, gamma, beta, out=inter)
        _check(x, 8, gamma, beta, 1e-6, "none", inter)
        same = x[:1].expand(3, 150, c)
        got = capi.group_norm(same, 8, gamma, beta)
        _check(same, 8, gamma, beta, 1e-6, "none", got)
        capi.group_norm(wide[:, :, :c], 8, gamma, beta, activation=capi.ACT_SILU, out=wide[:, :, :c])
        _check(x, 8, gamma, beta, 1e-6, "silu", wide[:, :, :c])
        assert (wide[:, :, c:] == 7).all()


@pytest.mark.parametrize("offset", [1e2, 1e4])
def test_means_far_from_zero(offset):
    """Means 100 and 10,000 deviations large: sums of squares alone would lose
    the variance."""
    import torch
    x, gamma, beta = _draw((2, 3000, 32), "float32", 5)
    x = x + offset
    got = capi.group_norm(x, 8, gamma, beta)
    _check(x, 8, gamma, beta, 1e-6, "none", got)


def test_constant_groups():
    """No deviation at all: beta, whatever the value."""
    import torch
    x = torch.full((2, 500, 24), 1234.5678, device="cuda")
    beta = torch.randn(24, device="cuda")
    got = capi.group_norm(x, 3, None, beta)
    assert torch.equal(got, beta.expand(2, 500, 24))


@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("pixels", [40, 9000])
def test_non_finite_values_stay_in_their_group(bad, pixels):
    import torch
    x, gamma, beta = _draw((3, pixels, 64), "bfloat16", 9)
    clean = capi.group_norm(x, 8, gamma, beta)
    x[1, pixels // 2, 20] = float(bad)   # group 2 of frame 1
    got = capi.group_norm(x, 8, gamma, beta)
    assert got[1, :, 16:24].isnan().all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[1, :, 16:24] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("y_type", TYPES)
@pytest.mark.parametrize("c,g", [(2, 1), (6, 2), (18, 9), (134, 2), (40, 5), (1030, 103)])
def test_rows_on_four_bytes_and_on_two(x_type, y_type, c, g):
    """Channels in pieces of two and more, rows that start anywhere."""
    import torch
    for p in (33, 2500):
        x, gamma, beta = _draw((2, p, c), x_type, c + p)
        plain = capi.group_norm(x, g, gamma, beta, 1e-6, capi.ACT_SILU, out_dtype=getattr(torch, y_type))
        _check(x, g, gamma, beta, 1e-6, "silu", plain)
        for pad, first in ((2, 2), (4, 2), (3, 1), (1, 0)):
            wide = torch.full((2, p, c + pad), float("nan"), dtype=x.dtype, device="cuda")
            wide[:, :, first:first + c] = x
            out = torch.full((2, p, c + pad), 5.0, dtype=plain.dtype, device="cuda")
            capi.group_norm(wide[:, :, first:first + c], g, gamma, beta, 1e-6, capi.ACT_SILU,
                            out=out[:, :, first:first + c])
            _check(x, g, gamma, beta, 1e-6, "silu", out[:, :, first:first + c])
            assert (out[:, :, :first] == 5).all() and (out[:, :, first + c:] == 5).all()


@pytest.mark.parametrize("pixels", [40, 9000, 200000])
def test_deviations_whose_squares_overflow_show(pixels):
    """Squares past fp32's range leave no plausible values: NaN, or zeros of an
    infinite variance; other groups stay as they are."""
    import torch
    x, _, _ = _draw((1, pixels, 32), "float32", 5)
    want = capi.group_norm(x, 4)
    x[:, :, 8:16] *= 1e25
    got = capi.group_norm(x, 4)
    bad = got[:, :, 8:16]
    assert (bad.isnan() | (bad == 0)).all()
    keep = [c for c in range(32) if not 8 <= c < 16]
    assert torch.equal(got[:, :, keep], want[:, :, keep])


def test_equal_parts_with_overflowing_squares_show():
    """The same when every part of the sums has one mean, so that none of the
    variance lies between parts: blocks of 64 pixels, zero and 1e25 in turn."""
    import torch
    p = 256 * 768
    x = torch.where((torch.arange(p, device="cuda") // 64) % 2 == 0, 0.0, 1e25)
    got = capi.group_norm(x[None, :, None].expand(1, p, 32).contiguous(), 4)
    assert (got.isnan() | (got == 0)).all()


def test_no_rows():
    import torch
    for shape in ((0, 5, 16), (2, 0, 16)):
        x = torch.empty(shape, device="cuda")
        assert capi.group_norm(x, 4).shape == shape


def test_repeats_streams_and_capture():
    """Bit for bit the same again, on another stream and replayed from a graph,
    with the program's own work in between."""
    import torch
    x, gamma, beta = _draw((2, 6000, 128), "bfloat16", 3)
    want = capi.group_norm(x, 32, gamma, beta, activation=capi.ACT_SILU)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = capi.group_norm(x, 32, gamma, beta, activation=capi.ACT_SILU)
    side.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = capi.group_norm(x, 32, gamma, beta, activation=capi.ACT_SILU)
    for i in range(3):
        x.copy_(_draw((2, 6000, 128), "bfloat16", 20 + i)[0])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, capi.group_norm(x, 32, gamma, beta, activation=capi.ACT_SILU))


def test_frames_far_apart():
    """Frame strides past 2^31 elements, pixel strides past 2^24."""
    import torch
    x, gamma, beta = _draw((3, 90, 64), "bfloat16", 11)
    for shape, strides in (((3, 90, 64), (2 ** 31 + 64, 64, 1)), ((3, 90, 64), (64, 2 ** 25, 1))):
        size = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
        big = [torch.empty(size, dtype=x.dtype, device="cuda").as_strided(shape, strides) for _ in range(2)]
        big[0].copy_(x)
        capi.group_norm(big[0], 8, gamma, beta, out=big[1])
        _check(x, 8, gamma, beta, 1e-6, "none", big[1])
        del big
    torch.cuda.empty_cache()


def test_more_pixels_than_24_bits():
    """One frame of 17 million pixels: counts that fp32 rounds, many chunks."""
    import torch
    x, gamma, beta = _draw((1, 17_000_003, 4), "float16", 12)
    got = capi.group_norm(x, 2, gamma, beta)
    _check(x, 2, gamma, beta, 1e-6, "none", got)


@pytest.mark.parametrize("act", ["gelu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("y_type", TYPES)
@pytest.mark.parametrize("pixels", [40, 30000])
def test_activations_of_infinities(act, y_type, pixels):
    """By a beta: +inf stays, a NaN too, -inf is -inf times 0, NaN."""
    import torch
    import row_operators as ro
    x, gamma, beta = _draw((2, pixels, 24), "float32", 8)
    beta[:8] = float("inf")
    beta[8:12] = float("-inf")
    beta[12:16] = float("nan")
    y = capi.group_norm(x, 3, gamma, beta, 1e-6, ro.ACTS[act], out_dtype=getattr(torch, y_type))
    assert (y[:, :, :8] == float("inf")).all()
    assert y[:, :, 8:16].isnan().all() and y[:, :, 16:].isfinite().all()


# one launch; single channels, 450 pixels a thread; vectors of four, 200; frames of
# 16-bit rows, vectors of eight, 112
@pytest.mark.parametrize("size", [(1, 64, 512, 32, "float32"), (2, 2000, 512, 32, "float32"),
                                  (1, 7000, 4, 1, "float32"), (1, 59_000_000, 1, 1, "float32"),
                                  (1, 26_214_400, 4, 1, "float32"), (4, 230400, 128, 32, "bfloat16")], ids=str)
@pytest.mark.parametrize("far", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("count", [1, 700])
def test_values_far_from_the_others(size, far, count):
    """The first value, or the first pixels (a border), far from all others, which are
    where the statistics begin."""
    import torch
    import row_operators as ro
    f, p, c, g, dtype = size
    gen = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn(f, p, c, generator=gen, device="cuda")
    if count == 1:
        x[:, 0, ::c // g] += far
    else:
        x[:, :min(count, p // 3)] += far
    x = x.to(getattr(torch, dtype))
    y = capi.group_norm(x, g, out_dtype=torch.float32)
    for i in range(f):
        want, bound = ro.group_norm_by_variance(x[i:i + 1], g, None, None, 1e-6, "none", y.dtype)
        ro.check(y[i:i + 1], want, bound)


@pytest.mark.parametrize("c", [4000, 4001])
@pytest.mark.parametrize("pixels", [3, 300])
def test_erf_gelu_of_fp32_results(c, pixels):
    """To fp32's precision relative to the value, out into the negative tail."""
    import torch
    import row_operators as ro
    beta = torch.linspace(-12, 12, c, device="cuda")
    for dtype in TYPES:
        x = torch.full((1, pixels, c), 3.0, dtype=getattr(torch, dtype), device="cuda")
        y = capi.group_norm(x, 1, None, beta, 1e-6, capi.ACT_GELU, out_dtype=torch.float32)
        v = beta.double().expand(1, pixels, c)
        ro.check(y, ro.exact_gelu(v), ro.exact_gelu_error(v))
