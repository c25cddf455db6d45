"""MXFP4 quantisation and products against float64."""
import pytest
import torch

import mx_cross as mc
import row_operators as ro
from seedvr2_ncnn_amd import capi

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rows(m, k, dtype, seed, pad=0, start=0):
    """Rows of blocks of very different sizes, `pad` elements between them."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen)
    x *= torch.exp2(torch.randint(-12, 8, (m, mc.blocks(k)), generator=gen).float()).repeat_interleave(32, 1)[:, :k]
    flat = torch.full((start + m * (k + pad),), 1e4, dtype=dtype, device="cuda")
    view = flat[start:].view(m, k + pad)[:, :k]
    view.copy_(x)
    return view


def _equal(rows, x):
    code, scale = mc.quantize(x)
    assert torch.equal(rows.scales.cpu().long(), scale.long())
    assert torch.equal(mc.unpack(rows.codes), code)
    return code, scale


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,pad,start", [
    (1, 1, 0, 0), (1, 31, 0, 0), (3, 32, 0, 0), (5, 33, 0, 0), (2, 1000, 8, 0), (7, 4097, 3, 1), (65, 8, 1, 3),
    (513, 2560, 0, 0), (300, 17, 0, 1), (1, 30001, 0, 5)])
def test_quantize(dtype, m, k, pad, start):
    x = _rows(m, k, dtype, m + k, pad, start)
    rows = capi.mx_quantize(x)
    code, scale = _equal(rows, x)
    for out_dtype in (dtype, torch.float32):
        got = capi.mx_dequantize(rows, out_dtype)
        assert torch.equal(got.double().cpu(), mc.values(code, scale, k))


def test_quantize_at_every_border():
    """Numbers, the middles between them and their neighbours, zeros of both signs."""
    edge = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    near = torch.cat([edge, torch.nextafter(edge, torch.tensor(9.0)),
                      torch.nextafter(edge, torch.tensor(-9.0))])
    near = torch.cat([near, -near])
    x = torch.zeros(len(near), 32)
    x[:, 0] = 4.0   # the scale is 1
    x[:, 5] = near
    x[:, 31] = -near
    _equal(capi.mx_quantize(x.cuda()), x)
    y = torch.zeros(64, 64)
    y[:, 0] = torch.linspace(4.0, 7.9999, 64)
    y[:, 33] = -torch.linspace(0.0, 1e-3, 64)
    _equal(capi.mx_quantize(y.cuda()), y)


def test_quantize_far_exponents():
    """The smallest and largest magnitudes of fp32, subnormals among them."""
    e = torch.arange(-149, 128)
    x = torch.zeros(len(e), 32)
    x[:, 0] = torch.ldexp(torch.ones(len(e)), e)
    x[:, 1] = -x[:, 0] * 0.30
    x[:, 2] = torch.where(e < 127, x[:, 0] * 1.9, x[:, 0])
    x[:, 3] = 2.0 ** -149
    rows = capi.mx_quantize(x.cuda())
    code, scale = _equal(rows, x)
    assert torch.equal(capi.mx_dequantize(rows, torch.float32).double().cpu(), mc.values(code, scale, 32))
    h = torch.zeros(26, 32, dtype=torch.float16)
    h[:, 0] = torch.ldexp(torch.ones(26), torch.arange(-24, 2)).half()
    h[:, 1] = -h[:, 0] * 0.75
    h[:, 7] = 2.0 ** -24
    rows = capi.mx_quantize(h.cuda())
    code, scale = _equal(rows, h)
    assert torch.equal(capi.mx_dequantize(rows, torch.float16).double().cpu(), mc.values(code, scale, 32))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_blocks_without_values_are_nan_and_no_others(dtype):
    x = torch.randn(6, 100).to(dtype)
    x[0, 3], x[1, 40], x[2, 99], x[3, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[5] = 0.0
    rows = capi.mx_quantize(x.cuda())
    _equal(rows, x)
    y = capi.mx_dequantize(rows, dtype)
    bad = torch.zeros(6, 100, dtype=torch.bool)
    bad[0, :32], bad[1, 32:64], bad[2, 96:], bad[3, 64:96] = True, True, True, True
    assert torch.equal(y.isnan().cpu(), bad)


def test_quantize_writes_whole_blocks_and_nothing_else():
    x = torch.randn(5, 70, device="cuda")
    codes = torch.full((7, 64), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((7, 9), 0xEE, dtype=torch.uint8, device="cuda")
    out = capi.MxRows(codes[1:6, :48], scales[1:6, 2:5], 70)
    assert capi.mx_quantize(x, out=out) is out
    _equal(out, x)
    assert (codes[0] == 0xEE).all() and (codes[6] == 0xEE).all() and (codes[:, 48:] == 0xEE).all()
    assert (scales[:, :2] == 0xEE).all() and (scales[:, 5:] == 0xEE).all() and (scales[::6] == 0xEE).all()
    wide = torch.full((6, 75), 7.0, dtype=torch.float16, device="cuda")
    capi.mx_dequantize(out, out=wide[:5, 1:71])
    assert (wide[5] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 71:] == 7).all()


def _weight(n, k, seed, stride=None):
    gen = torch.Generator().manual_seed(seed)
    code, scale = mc.quantize(torch.randn(n, k, generator=gen) * k ** -0.5 *
                              torch.exp2(torch.randint(-4, 4, (n, 1), generator=gen).float()))
    return capi.MxRows(*mc.pack(code, scale, stride=stride), k), mc.values(code, scale, k)


def _product(m, n, k, x_kind, y_dtype, act, with_bias, with_residual, seed=0, x_pad=0, y_pad=0, stride=None,
             **kwargs):
    gen = torch.Generator().manual_seed(1000 + seed)
    weight, w = _weight(n, k, seed, stride)
    rows = torch.randn(m, k, generator=gen)
    if x_kind is None:
        code, scale = mc.quantize(rows)
        x, xv = capi.MxRows(*mc.pack(code, scale, stride=stride), k), mc.values(code, scale, k)
    else:
        wide = torch.zeros(m, k + x_pad, dtype=x_kind)
        wide[:, :k] = rows
        x = wide.cuda()[:, :k]
        xv = wide[:, :k].double()
    bias = torch.randn(n, generator=gen) if with_bias else None
    wide = torch.randn(m, n + y_pad, generator=gen).to(y_dtype).cuda()
    residual = wide[:, :n] if with_residual else None
    out = torch.full((m, n + y_pad), 3.0, dtype=y_dtype, device="cuda")
    got = capi.mx_linear(x, weight, None if bias is None else bias.cuda(), ro.ACTS[act], residual, out=out[:, :n],
                         **kwargs)
    assert (out[:, n:] == 3).all()
    want, bound = mc.linear(xv.cuda(), w.cuda(), None if bias is None else bias.cuda(), act, residual, y_dtype)
    ro.check(got, want, bound)
    return x, weight, got


KINDS = [None] + TYPES


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 1000, 2560), (2, 17, 33), (16, 64, 256), (17, 100, 1000), (33, 48, 31), (64, 640, 512),
    (129, 65, 4096), (300, 513, 1001), (1000, 255, 96), (1, 7, 20000)])
def test_product(x_kind, m, n, k):
    _product(m, n, k, x_kind, torch.float32, "none", False, False, seed=m + n + k)


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("y_dtype", TYPES, ids=str)
@pytest.mark.parametrize("m", [3, 40, 515])
def test_product_epilogues(x_kind, y_dtype, m):
    for i, act in enumerate(ro.ACTS):
        _product(m, 130 + 2 * i, 640, x_kind, y_dtype, act, i != 1, i != 2, seed=i)


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m,n,k", [(5, 33, 100), (260, 129, 1000), (700, 512, 2048)])
def test_product_strides(x_kind, m, n, k):
    """Rows inside wider buffers; scales that start at 16 bytes, anywhere, close up."""
    for pad, y_pad, stride in ((3, 1, mc.blocks(k)), (8, 4, mc.blocks(k) + 5), (1, 7, None)):
        _product(m, n, k, x_kind, torch.bfloat16, "none", True, True, pad, pad, y_pad, stride)


@pytest.mark.parametrize("x_kind", [None, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m", [20, 600])
def test_product_without_workspace(x_kind, m):
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    _product(m, 300, 1500, x_kind, torch.float32, "gelu", True, True, workspace=none, stride=mc.blocks(1500) + 1)


@pytest.mark.parametrize("m,n,k", [(4096, 1024, 512), (2000, 3000, 256), (5000, 77, 2560), (90, 10240, 2560)])
def test_product_of_many_tiles(m, n, k):
    _product(m, n, k, None, torch.bfloat16, "silu", True, True)


def test_products_of_far_scales():
    """Blocks whose scales differ by 2^60 and lie near the ends of fp32's range."""
    gen = torch.Generator().manual_seed(3)
    for m in (4, 300):
        code = torch.randint(0, 16, (m, 256), generator=gen)
        xs = torch.randint(100, 160, (m, 8), generator=gen)
        wcode = torch.randint(0, 16, (96, 256), generator=gen)
        ws = torch.randint(60, 120, (96, 8), generator=gen)
        x, w = mc.values(code, xs, 256).cuda(), mc.values(wcode, ws, 256).cuda()
        got = capi.mx_linear(capi.MxRows(*mc.pack(code, xs), 256), capi.MxRows(*mc.pack(wcode, ws), 256),
                             out_dtype=torch.float32)
        ro.check(got, *mc.linear(x, w, None, "none", None, torch.float32))


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m,n", [(3, 96), (130, 96), (1500, 1000), (90, 2560)])
@pytest.mark.parametrize("low,high", [(0, 4), (0, 190), (180, 210)])
def test_weights_of_far_scales(x_kind, m, n, low, high):
    """Scales from the least one on, whose values are subnormal in bf16; sums that are normal."""
    gen = torch.Generator().manual_seed(4 + low + high)
    code, scale = torch.randint(0, 16, (n, 704), generator=gen), torch.randint(low, high, (n, 22), generator=gen)
    rows = (1 + torch.rand(m, 700, generator=gen)) * 1024
    w = mc.values(code, scale, 704)[:, :700]
    weight = capi.MxRows(*mc.pack(code, scale), 704)
    if x_kind is None:
        xcode, xscale = mc.quantize(torch.nn.functional.pad(rows, (0, 4)))
        x, xv = capi.MxRows(*mc.pack(xcode, xscale), 704), mc.values(xcode, xscale, 704)[:, :700]
    else:
        x = torch.nn.functional.pad(rows, (0, 4)).to(x_kind).cuda()
        xv = x[:, :700].double().cpu()
    got = capi.mx_linear(x, weight, out_dtype=torch.float32)
    ro.check(got, *mc.linear(xv.cuda(), w.cuda(), None, "none", None, torch.float32))


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m", [3, 300])
def test_nan_reaches_its_row_or_column_alone(x_kind, m):
    weight, _ = _weight(70, 320, 1)
    x = torch.randn(m, 320, device="cuda")
    x[1, 7] = float("nan")
    weight.scales[5, 9] = 255
    rows = capi.mx_quantize(x) if x_kind is None else x.to(x_kind)
    y = capi.mx_linear(rows, weight, out_dtype=torch.float32)
    bad = torch.zeros(m, 70, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 5] = True, True
    assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("x_kind", [None, torch.float32], ids=str)
@pytest.mark.parametrize("m", [3, 300])
def test_residual_in_place(x_kind, m):
    weight, w = _weight(96, 256, 2)
    rows = torch.randn(m, 256, device="cuda")
    x = capi.mx_quantize(rows) if x_kind is None else rows
    res = torch.randn(m, 96, device="cuda")
    want = capi.mx_linear(x, weight, residual=res, out_dtype=torch.float32)
    assert capi.mx_linear(x, weight, residual=res, out=res) is res
    assert torch.equal(res, want)


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m", [2, 100, 1030])
def test_graphs_and_streams(x_kind, m):
    """Two captured calls with workspaces of their own, replayed between eager work; equal
    every time."""
    weight, _ = _weight(200, 1024, 4)
    rows = [torch.randn(m, 1024, device="cuda").to(x_kind or torch.float32) for _ in range(2)]
    xs = [capi.mx_quantize(r) if x_kind is None else r for r in rows]
    want = [capi.mx_linear(x, weight, out_dtype=torch.float32) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = [torch.zeros(m, 200, device="cuda") for _ in xs]
    graphs = []
    for x, o in zip(xs, out):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            capi.mx_linear(x, weight, out=o)
        graphs.append(g)
    for _ in range(3):
        for g, o, w in zip(graphs, out, want):
            o.zero_()
            g.replay()
            assert torch.equal(capi.mx_linear(xs[0], weight, out_dtype=torch.float32), want[0])
            torch.cuda.synchronize()
            assert torch.equal(o, w)
    with torch.cuda.stream(side):
        y = capi.mx_linear(xs[1], weight, out_dtype=torch.float32)
    z = capi.mx_linear(xs[1], weight, out_dtype=torch.float32, stream=side)
    side.synchronize()
    assert torch.equal(y, want[1]) and torch.equal(z, want[1])


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
def test_calls_side_by_side(x_kind):
    """Two streams at once, each call with a workspace of its own."""
    weight, _ = _weight(300, 1500, 7, mc.blocks(1500) + 1)
    rows = [torch.randn(m, 1500, device="cuda").to(x_kind or torch.float32) for m in (90, 700)]
    xs = [capi.mx_quantize(r) if x_kind is None else r for r in rows]
    want = [capi.mx_linear(x, weight, out_dtype=torch.float32) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, x in enumerate(xs):
            got[i].append(capi.mx_linear(x, weight, out_dtype=torch.float32, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("x_kind", KINDS[1:], ids=str)
def test_rows_that_begin_anywhere(x_kind):
    """Single elements past 16 bytes, odd strides; few rows and many."""
    weight, w = _weight(50, 333, 8)
    for m in (2, 20, 600):
        flat = torch.randn(1 + m * 335, device="cuda").to(x_kind)
        x = flat[1:].view(m, 335)[:, :333]
        got = capi.mx_linear(x, weight, out_dtype=torch.float32)
        ro.check(got, *mc.linear(x.double(), w.cuda(), None, "none", None, torch.float32))


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
def test_broadcast_row(x_kind):
    """Many equal rows, and an out whose rows lie far apart."""
    weight, w = _weight(40, 256, 9)
    row = torch.randn(1, 256, device="cuda").to(x_kind or torch.float32)
    x = row.repeat(70, 1)
    x = capi.mx_quantize(x) if x_kind is None else x
    far = torch.zeros(70, 1 << 16, device="cuda")
    got = capi.mx_linear(x, weight, out=far[:, 7:47])
    assert torch.equal(got, got[:1].expand(70, 40)) and far.count_nonzero() == got.count_nonzero()


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m", [9, 16, 17])
def test_wide_weight(x_kind, m):
    """64 columns a workgroup, and as much of x as they hold at once."""
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    _product(m, 12300, 2600, x_kind, torch.float32, "none", False, False, workspace=none)


@pytest.mark.parametrize("x_kind", [None, torch.bfloat16], ids=str)
def test_more_tiles_than_a_launch_has(x_kind):
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    weight, _ = _weight(8192, 32, 10, stride=17)   # (scales that tiles would copy)
    m, some = (1 << 20) + 20, 37
    x = torch.randn(some, 32, device="cuda").bfloat16()
    rows = x.repeat((m + some - 1) // some, 1)[:m]
    first = capi.mx_linear(capi.mx_quantize(x) if x_kind is None else x, weight, workspace=none)
    got = capi.mx_linear(capi.mx_quantize(rows) if x_kind is None else rows, weight, workspace=none)
    whole = m // some * some
    assert (got[:whole].view(-1, some, 8192) == first).all() and torch.equal(got[whole:], first[:m - whole])


@pytest.mark.parametrize("x_kind", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(40, 200, 3000), (65, 513, 264), (129, 2560, 1000), (300, 130, 72), (200, 1543, 8)])
def test_codes_on_tiles(x_kind, m, n, k):
    """Rows of other types on tiles of the weight's codes: steps, planes and ranges that end early."""
    _product(m, n, k, x_kind, torch.float16, "gelu", True, True, seed=m)
    _product(m, n, k, x_kind, torch.float32, "none", False, False, seed=k, stride=mc.blocks(k) + 1)


def test_mlp_in_four_bits():
    """Quantise, product with GELU, quantise, product onto the residual, as an MLP runs them:
    every step against float64 on its own inputs."""
    x = torch.randn(333, 320, device="cuda")
    up, w0 = _weight(640, 320, 5)
    down, w1 = _weight(320, 640, 6)
    xq = capi.mx_quantize(x)
    h = capi.mx_linear(xq, up, activation=capi.ACT_GELU)
    hq = capi.mx_quantize(h)
    y = capi.mx_linear(hq, down, residual=x, out_dtype=torch.float32)
    code, scale = mc.quantize(x)
    ro.check(h, *mc.linear(mc.values(code, scale, 320).cuda(), w0.cuda(), None, "gelu", None, torch.bfloat16))
    code, scale = mc.quantize(h)
    ro.check(y, *mc.linear(mc.values(code, scale, 640).cuda(), w1.cuda(), None, "none", x, torch.float32))


def _codes(rows, k, gen, low, high, stride=None):
    """Random codes under scales low .. high - 1 that differ from block to block: (MxRows, values)."""
    b = mc.blocks(k)
    code = torch.randint(0, 16, (rows, 32 * b), generator=gen)
    code[:, k:] = 0
    scale = torch.randint(low, high, (rows, b), generator=gen)
    return capi.MxRows(*mc.pack(code, scale, stride=stride), k), mc.values(code, scale, k)


def _dealt_bytes(m, n, k):
    """What the scales of 256 x 256 tiles take: 1 KB for 128 rows of x and 256 k, 512 bytes
    for 64 rows of the weight."""
    steps = (mc.blocks(k) + 7) // 8
    return ((m + 255) // 256 * 2 * 1024 + (n + 255) // 256 * 4 * 512) * steps


@pytest.mark.parametrize("y_dtype,act,epilogue", [
    (torch.float32, "none", False), (torch.bfloat16, "gelu", True), (torch.float16, "silu", True),
    (torch.float32, "gelu_tanh", True)], ids=str)
@pytest.mark.parametrize("m,n,k,stride", [
    (3841, 4000, 1500, None), (4090, 4090, 1700, 55), (2047, 8191, 1600, 50), (3900, 4001, 520, None)])
def test_largest_tiles(m, n, k, stride, y_dtype, act, epilogue):
    """256 x 256 tiles that end in rows, columns and k; two steps of 256 k and more, the stages
    filled again; equal every time."""
    assert capi.mx_linear_workspace(m, n, k) == (_dealt_bytes(m, n, k) + 255) // 256 * 256
    gen = torch.Generator().manual_seed(m + k)
    x, xv = _codes(m, k, gen, 117, 130, stride)
    weight, w = _codes(n, k, gen, 113, 125, stride)
    bias = torch.randn(n, generator=gen).cuda() if epilogue else None
    residual = torch.randn(m, n, generator=gen).to(y_dtype).cuda() if epilogue else None
    got = capi.mx_linear(x, weight, bias, ro.ACTS[act], residual, out_dtype=y_dtype)
    ro.check(got, *mc.linear(xv.cuda(), w.cuda(), bias, act, residual, y_dtype))
    for _ in range(3):
        assert torch.equal(capi.mx_linear(x, weight, bias, ro.ACTS[act], residual, out_dtype=y_dtype), got)


@pytest.mark.parametrize("stride", [None, 1000], ids=str)
@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m,n,k", [
    (17, 320, 20000), (64, 64, 10240), (200, 2560, 10240), (77, 2560, 5120), (40, 200, 2560), (300, 5120, 2560),
    (1000, 1000, 9000), (2000, 2000, 8192), (4096, 4096, 2560)])
def test_queried_workspace_is_what_a_larger_one_gives(m, n, k, x_kind, stride):
    """The same tiles and ranges of k, and so the same sums to the bit."""
    gen = torch.Generator().manual_seed(n)
    weight, _ = _codes(n, k, gen, 113, 125, stride)
    if x_kind is None:
        x, _ = _codes(m, k, gen, 117, 130, stride)
        kind = None
    else:
        x = torch.randn(m, k, generator=gen).to(x_kind).cuda()
        kind = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16, torch.float16: capi.DTYPE_F16}[x_kind]
    size = capi.mx_linear_workspace(m, n, k, kind, capi.DTYPE_F32)
    queried, more = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (size, size + (1 << 30)))
    a = capi.mx_linear(x, weight, out_dtype=torch.float32, workspace=queried)
    assert torch.equal(a, capi.mx_linear(x, weight, out_dtype=torch.float32, workspace=more))


@pytest.mark.parametrize("m", [1, 3])
@pytest.mark.parametrize("x_kind", [None, torch.bfloat16], ids=str)
def test_more_columns_than_a_launch_has(x_kind, m):
    some, n = 37, (1 << 29) + 100
    times = (n + some - 1) // some
    gen = torch.Generator().manual_seed(18)
    few, _ = _codes(some, 32, gen, 113, 125)
    weight = capi.MxRows(few.codes.repeat(times, 1)[:n], few.scales.repeat(times, 1)[:n], 32)
    x = torch.randn(m, 32, generator=gen).bfloat16().cuda()
    if x_kind is None:
        x = capi.mx_quantize(x)
    bias = torch.randn(some, generator=gen).cuda()
    residual = torch.randn(m, some, generator=gen).bfloat16().cuda()
    first = capi.mx_linear(x, few, bias, capi.ACT_SILU, residual)
    out = residual.repeat(1, times)[:, :n]
    capi.mx_linear(x, weight, bias.repeat(times)[:n], capi.ACT_SILU, out, out=out)
    whole = n // some * some
    assert (out[:, :whole].view(m, -1, some) == first[:, None]).all()
    assert torch.equal(out[:, whole:], first[:, :n - whole])


def test_more_tiles_of_codes_than_a_launch_has():
    """Many rows on the weight's codes, which take no workspace."""
    some, m, n, k = 37, (1 << 29) + 100, 17, 8
    gen = torch.Generator().manual_seed(19)
    weight, _ = _codes(n, k, gen, 113, 125, 16)
    x = torch.randn(some, k, generator=gen).bfloat16().cuda()
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    first = capi.mx_linear(x, weight, workspace=none)
    got = capi.mx_linear(x.repeat((m + some - 1) // some, 1)[:m], weight, workspace=none)
    whole = m // some * some
    assert (got[:whole].view(-1, some, n) == first).all() and torch.equal(got[whole:], first[:m - whole])


@pytest.mark.parametrize("m,n", [(3, 96), (16, 2560), (130, 96), (700, 2560), (3000, 2560)])
@pytest.mark.parametrize("exponent", [-100, -112, -120, -126, -140])
def test_fp32_rows_near_the_smallest_numbers(m, n, exponent):
    """Three bf16 terms hold a value to within half of bf16's smallest number, 2^-134, which large
    weights bring to light."""
    gen = torch.Generator().manual_seed(m - exponent)
    weight, w = _codes(n, 320, gen, 220, 240)
    x = torch.ldexp(torch.randn(m, 320, generator=gen, dtype=torch.float64), torch.tensor(exponent)).float()
    got = capi.mx_linear(x.cuda(), weight)
    want, bound = mc.linear(x.double().cuda(), w.cuda(), None, "none", None, torch.float32)
    ro.check(got, want, bound + 2.0 ** -134 * w.abs().sum(dim=1).cuda())


@pytest.mark.parametrize("x_kind", KINDS, ids=str)
@pytest.mark.parametrize("m", [3, 300])
def test_weights_past_the_largest_number_reach_their_column_alone(x_kind, m):
    gen = torch.Generator().manual_seed(m)
    weight, w = _codes(70, 320, gen, 113, 125)
    x, xv = _codes(m, 320, gen, 117, 130)
    if x_kind is not None:
        x = xv.to(x_kind).cuda()   # (six of 2^2 at most, four bits)
    weight.scales[5, 3] = 254
    weight.codes[5, 3 * 16:4 * 16] = 0x77
    got = capi.mx_linear(x, weight, out_dtype=torch.float32)
    want, bound = mc.linear(xv.cuda(), w.cuda(), None, "none", None, torch.float32)
    keep = torch.arange(70, device="cuda") != 5
    ro.check(got[:, keep], want[:, keep], bound[:, keep])
