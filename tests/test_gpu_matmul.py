"""s2_linear and s2_grouped_linear against a float64 form: types, sizes from one
row, column and product to many tiles, strides, alignment, residuals in place,
ragged and empty groups, rows outside them, and non-finite values."""
import pytest

from seedvr2_ncnn_amd import capi

pytestmark = pytest.mark.gpu

# x, weight
PAIRS = [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float16")]
Y_TYPES = ["float32", "bfloat16", "float16"]
# (m, k, n): single ones; k below, at and past a k-step and of no even alignment;
# n that ends inside a 16-column piece, a wave's and a tile's columns; row counts
# around 16, 64, 128 and 256
SIZES = [(1, 1, 1), (1, 2560, 130), (2, 7, 16), (3, 132, 300), (15, 33, 17), (16, 64, 64),
         (17, 72, 48), (33, 129, 257), (64, 1000, 129), (65, 192, 512), (127, 8, 8), (129, 320, 100),
         (255, 640, 264), (257, 65, 128), (300, 2048, 256), (520, 96, 1030)]


# enough tiles of 256 x 256 for every compute unit; one to six k steps, the last one
# ragged or not
MANY_TILES = [(4900, 64, 2560), (5001, 200, 2564), (3100, 328, 4104)]


def _gen(seed):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=gen, device="cuda")


def _operands(m, k, n, pair, y_type, groups=0, seed=0):
    import torch
    draw = _gen(seed + m + 7 * k + n)
    x = draw(m, k).to(getattr(torch, pair[0]))
    lead = (groups,) if groups else ()
    w = (draw(*lead, n, k) * k ** -0.5).to(getattr(torch, pair[1]))
    bias = draw(*lead, n)
    res = draw(m, n).to(getattr(torch, y_type))
    return x, w, bias, res


def _check(got, x, w, bias, act, res):
    import row_operators as ro
    want, bound = ro.linear(x, w, bias, act, res, got.dtype)
    ro.check(got, want, bound)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_sizes(size, pair):
    import torch
    m, k, n = size
    x, w, bias, res = _operands(m, k, n, pair, "float32")
    got = capi.linear(x, w, bias, residual=res, out_dtype=torch.float32)
    _check(got, x, w, bias, "none", res)


@pytest.mark.parametrize("size", MANY_TILES, ids=str)
@pytest.mark.parametrize("y_type", Y_TYPES)
def test_many_tiles(size, y_type):
    import torch
    import row_operators as ro
    m, k, n = size
    for pair in PAIRS[1:]:
        x, w, bias, res = _operands(m, k, n, pair, y_type)
        for act, r in (("gelu", None), ("none", res), ("gelu_tanh", res)):
            got = capi.linear(x, w, bias, ro.ACTS[act], r, out_dtype=getattr(torch, y_type))
            _check(got, x, w, bias, act, r)


@pytest.mark.parametrize("size", [(1, 512, 160), (40, 256, 96), (200, 384, 272), (130, 100, 77)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("y_type", Y_TYPES)
def test_types_activations_and_residuals(size, pair, y_type):
    import torch
    import row_operators as ro
    m, k, n = size
    x, w, bias, res = _operands(m, k, n, pair, y_type)
    for act, code in ro.ACTS.items():
        for b, r in ((bias, None), (None, res), (bias, res)):
            got = capi.linear(x, w, b, code, r, out_dtype=getattr(torch, y_type))
            _check(got, x, w, b, act, r)


@pytest.mark.parametrize("m", [1, 48, 96, 300])
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("pads", [(8, 8, 8), (4, 12, 4), (1, 3, 5)], ids=str)
def test_strides_and_in_place(m, pair, pads):
    """Rows inside wider buffers at aligned and odd places; the residual as the
    output; nothing outside the output's rows and columns changes."""
    import torch
    k, n = 320, 136
    y_type = pair[0]
    x, w, bias, res = _operands(m, k, n, pair, y_type)
    px, pr, py = pads
    xw = torch.full((m, k + px), float("nan"), dtype=x.dtype, device="cuda")
    xw[:, px:] = x
    rw = torch.full((m, n + pr), float("nan"), dtype=res.dtype, device="cuda")
    rw[:, pr:] = res
    yw = torch.full((m + 2, n + 2 * py), 5.0, dtype=res.dtype, device="cuda")
    got = capi.linear(xw[:, px:], w, bias, capi.ACT_SILU, rw[:, pr:], out=yw[1:m + 1, py:py + n])
    _check(got, x, w, bias, "silu", res)
    inside = torch.zeros_like(yw, dtype=torch.bool)
    inside[1:m + 1, py:py + n] = True
    assert (yw[~inside] == 5).all()
    capi.linear(xw[:, px:], w, bias, capi.ACT_SILU, rw[:, pr:], out=rw[:, pr:])
    assert torch.equal(rw[:, pr:], got) and rw[:, :pr].isnan().all()


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_weights_at_odd_places(pair):
    """Weight and bias that start at no 16-byte boundary."""
    import torch
    for m in (2, 90, 300):
        x, w, bias, res = _operands(m, 256, 128, pair, "float32")
        wide = torch.empty(w.numel() + 3, dtype=w.dtype, device="cuda")
        odd = wide[3:].view_as(w)
        odd.copy_(w)
        wb = torch.empty(129, device="cuda")
        wb[1:] = bias
        got = capi.linear(x, odd, wb[1:], residual=res, out_dtype=torch.float32)
        _check(got, x, w, bias, "none", res)


@pytest.mark.parametrize("m,k,n", [(1, 512, 100), (60, 520, 64), (200, 4096, 130), (300, 132, 257)])
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_non_finite_values_stay_in_their_row(m, k, n, pair):
    """An infinity and a NaN in a row of x, a NaN in a residual: the row (the
    element) becomes non-finite, the others keep their bits; so do a column's
    neighbours of an infinite weight."""
    import torch
    x, w, bias, res = _operands(m, k, n, pair, "float32")
    clean = capi.linear(x, w, bias, residual=res, out_dtype=torch.float32)
    x[0, k // 2] = float("inf")
    x[m - 1, k - 1] = float("nan")
    res[m // 2, n - 1] = float("nan")
    got = capi.linear(x, w, bias, residual=res, out_dtype=torch.float32)
    assert not got[0].isfinite().any() and got[m - 1].isnan().all() and got[m // 2, n - 1].isnan()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[0] = keep[m - 1] = False
    keep[m // 2, n - 1] = False
    assert torch.equal(got[keep], clean[keep])
    x, w, bias, res = _operands(m, k, n, pair, "float32")
    w[n // 2, 3] = float("-inf")
    got = capi.linear(x, w, bias, residual=res, out_dtype=torch.float32)
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[:, n // 2] = False
    assert not got[:, n // 2].isfinite().any() and torch.equal(got[keep], clean[keep])


def test_large_fp32_values():
    """fp32 rows at the type's largest values and with 24-bit significands: taken
    exactly where y is fp32."""
    import torch
    x = torch.full((5, 64), torch.finfo(torch.float32).max, device="cuda")
    w = torch.zeros(32, 64, dtype=torch.bfloat16, device="cuda")
    w[torch.arange(32), torch.arange(32)] = 1.0
    got = capi.linear(x, w)
    assert torch.equal(got, x[:, :32])
    x = torch.randn(300, 64, device="cuda")
    assert torch.equal(capi.linear(x, w), x[:, :32])
    assert torch.equal(capi.linear(x[:3], w), x[:3, :32])


@pytest.mark.parametrize("m,k,n", [(77, 5120, 256), (130, 2560, 300), (257, 1024, 520)])
def test_with_and_without_workspace(m, k, n):
    """Split along k or not: both within the bound, each the same again."""
    import torch
    x, w, bias, res = _operands(m, k, n, PAIRS[1], "float32")
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    for ws in (None, none):
        got = capi.linear(x, w, bias, capi.ACT_GELU, res, out_dtype=torch.float32, workspace=ws)
        _check(got, x, w, bias, "gelu", res)
        again = capi.linear(x, w, bias, capi.ACT_GELU, res, out_dtype=torch.float32, workspace=ws)
        assert torch.equal(got, again)


# many fp32 rows of short k: k in one to five steps of 32, whole quads of it or not;
# rows and columns in and out of whole tiles
SHORT_K = [(2500, 132, 2564, "bfloat16"), (2601, 4, 2561, "bfloat16"), (20001, 96, 330, "float16"),
           (6300, 160, 1088, "float16"), (3333, 100, 2000, "bfloat16"), (2500, 96, 2564, "float32"),
           (25000, 36, 257, "float32"), (110000, 64, 60, "float32"), (2500, 133, 2564, "bfloat16"),
           (7001, 1, 1000, "float16"), (6300, 158, 1088, "bfloat16"), (2500, 95, 2563, "float32")]


@pytest.mark.parametrize("size", SHORT_K, ids=str)
def test_short_k(size):
    """Rows inside wider ones, a residual in place, every activation; an infinity and a
    NaN stay in their rows; one set of bits whatever the workspace."""
    import torch
    import row_operators as ro
    m, k, n, y_type = size
    x, w, bias, res = _operands(m, k, n, PAIRS[0], y_type)
    wide = torch.full((m, k + 8), float("nan"), device="cuda")
    wide[:, 4:4 + k] = x
    view = wide[:, 4:4 + k]
    for act, b, r in (("none", bias, None), ("gelu", None, res), ("silu", bias, res),
                      ("gelu_tanh", bias, None)):
        got = capi.linear(view, w, b, ro.ACTS[act], r, out_dtype=res.dtype)
        _check(got, x, w, b, act, r)
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    assert torch.equal(got, capi.linear(x, w, bias, ro.ACTS["gelu_tanh"], out_dtype=res.dtype,
                                        workspace=none))
    out = torch.full((m + 2, n + 4), 5.0, dtype=res.dtype, device="cuda")
    out[1:m + 1, 4:] = res
    inner = out[1:m + 1, 4:]
    want = capi.linear(x, w, bias, capi.ACT_SILU, res, out_dtype=res.dtype)
    capi.linear(x, w, bias, capi.ACT_SILU, inner, out=inner)
    assert torch.equal(inner, want)
    assert (out[0] == 5).all() and (out[-1] == 5).all() and (out[:, :4] == 5).all()
    plain = capi.linear(x, w, out_dtype=res.dtype)
    view[7, 0], view[m - 1, k - 1] = float("inf"), float("nan")
    bad = capi.linear(view, w, out_dtype=res.dtype)
    good = [i for i in range(m) if i not in (7, m - 1)]
    assert torch.equal(bad[good], plain[good])
    assert not bad[7].isfinite().any() and bad[m - 1].isnan().all()


# k, n and strides of every parity, so that rows begin anywhere; few rows and tiles
@pytest.mark.parametrize("m", [1, 17, 32, 70, 300])
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("kn", [(5001, 67), (515, 130), (262, 129), (1023, 258)], ids=str)
def test_rows_that_begin_anywhere(m, pair, kn):
    import torch
    k, n = kn
    x, w, bias, res = _operands(m, k, n, pair, "float16" if pair[0] == "float16" else "bfloat16")
    for first, pad in ((0, 0), (1, 2), (2, 3), (3, 6)):
        wide = torch.full((m, first + k + pad), float("nan"), dtype=x.dtype, device="cuda")
        wide[:, first:first + k] = x
        flat = torch.full((first + n * k + 9,), float("nan"), dtype=w.dtype, device="cuda")
        odd = flat[first:first + n * k].view(n, k)
        odd.copy_(w)
        out = torch.full((m + 1, first + n + pad), 5.0, dtype=res.dtype, device="cuda")
        inner = out[:m, first:first + n]
        inner.copy_(res)
        capi.linear(wide[:, first:first + k], odd, bias, capi.ACT_NONE, inner, out=inner)
        _check(inner, x, w, bias, "none", res)
        assert (out[m] == 5).all() and (out[:, :first] == 5).all() and (out[:, first + n:] == 5).all()


# above 32 rows; k and n even and odd; tiles beside and below each other
@pytest.mark.parametrize("size", [(33, 72, 48), (130, 100, 77), (129, 1000, 260), (300, 33, 513)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("y_type", Y_TYPES)
def test_sizes_without_workspace(size, pair, y_type):
    import torch
    m, k, n = size
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    x, w, bias, res = _operands(m, k, n, pair, y_type)
    got = capi.linear(x, w, bias, capi.ACT_SILU, res, out_dtype=res.dtype, workspace=none)
    _check(got, x, w, bias, "silu", res)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("kn", [(72, 33), (130, 260)], ids=str)
def test_groups_without_workspace(pair, kn):
    """Ragged and empty groups; rows in none keep what the output holds."""
    import torch
    k, n = kn
    starts = [3, 3, 150, 151, 400]
    x, w, bias, res = _operands(410, k, n, pair, pair[0], groups=4)
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    out = torch.full((410, n), 5.0, dtype=res.dtype, device="cuda")
    capi.grouped_linear(x, torch.tensor(starts, dtype=torch.int32, device="cuda"), w, bias,
                        capi.ACT_GELU, res, out=out, workspace=none)
    for g in range(4):
        at = slice(starts[g], starts[g + 1])
        if starts[g] < starts[g + 1]:
            _check(out[at], x[at], w[g], bias[g], "gelu", res[at])
    assert (out[:3] == 5).all() and (out[400:] == 5).all()


GROUPS = [[5], [0, 3, 0], [1] * 9, [130, 0, 1, 64, 0, 0, 257], [0] * 70 + [20, 0, 33], [16] * 40,
          [700, 2]]
# the same with enough 256 x 256 tiles for every compute unit
MANY_ROWS = [4000, 0, 255, 1, 0, 600]


@pytest.mark.parametrize("rows", GROUPS, ids=lambda r: "-".join(map(str, r[-5:])))
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("kn", [(256, 136), (72, 33), (1000, 260)], ids=str)
def test_groups(rows, pair, kn):
    _groups(rows, pair, kn)


@pytest.mark.parametrize("pair", PAIRS[1:], ids="-".join)
def test_groups_of_many_tiles(pair):
    _groups(MANY_ROWS, pair, (136, 2560))


def _groups(rows, pair, kn):
    """Rows before the first group and behind the last one keep what they held."""
    import torch
    import row_operators as ro
    k, n = kn
    before, behind = 3, 5
    m = before + sum(rows) + behind
    x, w, bias, res = _operands(m, k, n, pair, "float32", len(rows))
    x[:before] = float("nan")
    x[m - behind:] = float("inf")
    ends = [before]
    for r in rows:
        ends.append(ends[-1] + r)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    out = torch.full((m, n), 9.0, device="cuda")
    capi.grouped_linear(x, offsets, w, bias, capi.ACT_GELU_TANH, res, out=out)
    for g, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        if a < b:
            _check(out[a:b], x[a:b], w[g], bias[g], "gelu_tanh", res[a:b])
    assert (out[:before] == 9).all() and (out[m - behind:] == 9).all()
    got = capi.grouped_linear(x, offsets, w, out_dtype=torch.bfloat16)
    a = next(g for g, r in enumerate(rows) if r)
    _check(got[ends[a]:ends[a + 1]], x[ends[a]:ends[a + 1]], w[a], None, "none", None)


def test_offsets_out_of_range_are_clamped():
    """Offsets below 0 and past m stand for 0 and m; descending ones leave every
    byte outside y alone."""
    import torch
    x, w, bias, res = _operands(90, 128, 64, PAIRS[1], "float32", 3)
    whole = torch.full((94, 64), 2.0, device="cuda")
    out = whole[2:92]
    offs = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    capi.grouped_linear(x, offs(-7, 30, 60, 2 ** 31 - 1), w, bias, out=out)
    for g in range(3):
        _check(out[30 * g:30 * g + 30], x[30 * g:30 * g + 30], w[g], bias[g], "none", None)
    capi.grouped_linear(x, offs(80, 10, 200, -5), w, bias, out=out)
    torch.cuda.synchronize()
    assert (whole[:2] == 2).all() and (whole[92:] == 2).all()


def test_no_rows_and_no_groups():
    import torch
    w = torch.zeros(24, 16, dtype=torch.bfloat16, device="cuda")
    x = torch.empty(0, 16, dtype=torch.bfloat16, device="cuda")
    assert capi.linear(x, w).shape == (0, 24)
    offs = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert capi.grouped_linear(x, offs, w.expand(2, 24, 16).contiguous()).shape == (0, 24)
    out = torch.ones(4, 24, dtype=torch.bfloat16, device="cuda")
    rows = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")
    capi.grouped_linear(rows, offs[:1], w[None][:0], out=out)
    capi.grouped_linear(rows, offs, w.expand(2, 24, 16).contiguous(), out=out)
    torch.cuda.synchronize()
    assert (out == 1).all()


def test_repeats_streams_and_capture():
    import torch
    x, w, bias, res = _operands(300, 1280, 256, PAIRS[1], "bfloat16")
    _, wg, bg, _ = _operands(300, 1280, 256, PAIRS[1], "bfloat16", 3)
    offsets = torch.tensor([0, 100, 100, 290], dtype=torch.int32, device="cuda")

    def both():
        y = capi.linear(x, w, bias, capi.ACT_SILU, res)
        z = torch.zeros_like(y)
        return y, capi.grouped_linear(x, offsets, wg, bg, capi.ACT_GELU, res, out=z)

    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(3):
        x.copy_(_gen(40 + i)(300, 1280))
        offsets.copy_(torch.tensor([i, 90 + i, 120, 300], dtype=torch.int32))
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both()):
            assert torch.equal(a, b)


def test_timestep_embedding_chain():
    """Two timesteps to a block's modulation rows as the DiT's frontend does:
    embedding, product + SiLU, product + SiLU, product; fp32 rows, bf16 weights."""
    import torch
    import row_operators as ro
    draw = _gen(2)
    ws = [(draw(n, k) * k ** -0.5).bfloat16() for n, k in ((640, 256), (640, 640), (3840, 640))]
    bs = [0.1 * draw(w.shape[0]) for w in ws]
    h = capi.timestep_embedding([999.0, 0.5])
    for w, b, act in zip(ws, bs, ("silu", "silu", "none")):
        got = capi.linear(h, w, b, ro.ACTS[act])
        _check(got, h, w, b, act, None)
        h = got
    assert h.shape == (2, 3840)


def test_vae_attention_block():
    """The VAE's mid block on channels-last rows: group norm into VAEChunkedMHA, then
    x's 1x1x1 shortcut with the attention's output as its residual, in place; each
    step of this library against float64 on what went into it."""
    import torch
    import row_operators as ro
    draw = _gen(4)
    seq, c = 330, 128
    x = draw(1, seq, c).bfloat16()
    gamma, beta = 1 + 0.1 * draw(c), 0.1 * draw(c)
    h = capi.group_norm(x, 32, gamma, beta)
    ro.check(h, *ro.group_norm(x, 32, gamma, beta, 1e-6, "none", h.dtype))
    mats = [draw(c, c) * c ** -0.5 for _ in range(4)]
    zero = torch.zeros(c, device="cuda")
    mha = capi.Mha(1, *(t for w in mats for t in (w, zero)), scale=c ** -0.5)
    a = mha.forward(h[0])
    q, k, v = (h[0].float() @ w.t() for w in mats[:3])
    ref = torch.softmax(q @ k.t() * c ** -0.5, dim=-1) @ v @ mats[3].t()
    # bf16 projections, weights and sums: a few of their half steps
    assert ((a.float() - ref).norm() / ref.norm()).item() < 6 * 2.0 ** -8
    w, b = (draw(c, c) * c ** -0.5).bfloat16(), 0.1 * draw(c)
    before = a.clone()
    y = capi.linear(x[0], w, b, residual=a, out=a)
    _check(y, x[0], w, b, "none", before)


def test_two_stream_mlp():
    """A DiT block's MLP whose video and text rows have weights of their own, onto
    the fp32 residual stream in place."""
    import torch
    draw = _gen(6)
    rows, hidden, inner = [450, 64], 256, 1024
    m = sum(rows)
    offs = torch.tensor([0, rows[0], m], dtype=torch.int32, device="cuda")
    up = (draw(2, inner, hidden) * hidden ** -0.5).bfloat16()
    down = (draw(2, hidden, inner) * inner ** -0.5).bfloat16()
    bu, bd = 0.1 * draw(2, inner), 0.1 * draw(2, hidden)
    x, res = draw(m, hidden).bfloat16(), draw(m, hidden)
    start = res.clone()
    h = capi.grouped_linear(x, offs, up, bu, capi.ACT_GELU_TANH)
    capi.grouped_linear(h, offs, down, bd, residual=res, out=res)
    for g, (a, b) in enumerate(((0, rows[0]), (rows[0], m))):
        _check(h[a:b], x[a:b], up[g], bu[g], "gelu_tanh", None)
        _check(res[a:b], h[a:b], down[g], bd[g], "none", start[a:b])


def test_rows_far_apart():
    """Row strides whose offsets pass 32 bits within a tile and over the call: x, the
    residual and y each spread over 4.7 GB."""
    import torch
    m, k, n, far = 70, 72, 40, 2 ** 25 + 8
    for pair in PAIRS[1:]:
        x, w, bias, res = _operands(m, k, n, pair, pair[0])
        spread = [torch.empty(m * far, dtype=x.dtype, device="cuda") for _ in range(3)]
        xw, rw, yw = (t.as_strided((m, c), (far, 1)) for t, c in zip(spread, (k, n, n)))
        xw.copy_(x)
        rw.copy_(res)
        for args in ((xw, res, None), (x, res, yw), (x, rw, None), (xw, rw, rw)):
            got = capi.linear(args[0], w, bias, capi.ACT_SILU, args[1], out=args[2])
            _check(got, x, w, bias, "silu", res)
        del spread, xw, rw, yw
    torch.cuda.empty_cache()


def test_groups_whose_weights_pass_32_bits():
    """Three weights of 2^30 elements: the last one starts 4.3 GB in."""
    import torch
    n = k = 2 ** 15
    draw = _gen(7)
    w = torch.empty(3, n, k, dtype=torch.bfloat16, device="cuda")
    for part in w.view(-1, 2 ** 12, k):
        part.copy_(draw(2 ** 12, k) * k ** -0.5)
    for rows in ([1, 0, 2], [100, 3, 70]):
        ends = [0, rows[0], rows[0] + rows[1], sum(rows)]
        x = draw(ends[-1], k).bfloat16()
        got = capi.grouped_linear(x, torch.tensor(ends, dtype=torch.int32, device="cuda"), w,
                                  out_dtype=torch.float32)
        for g in (0, 2):
            for cols in (slice(0, 64), slice(n - 64, n)):
                _check(got[ends[g]:ends[g + 1], cols], x[ends[g]:ends[g + 1]], w[g, cols], None, "none", None)
    del w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [5, 90, 400])
def test_a_stream_that_is_not_the_current_one(m):
    """stream= with outputs and workspaces made by the call, while the current stream
    keeps taking and giving back memory of the same sizes."""
    import torch
    x, w, bias, res = _operands(m, 2560, 640, PAIRS[0], "float32")
    frames = x.view(1, m, 2560)
    want = capi.linear(x, w, bias, capi.ACT_SILU, res), capi.group_norm(frames, 32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        got.append((capi.linear(x, w, bias, capi.ACT_SILU, res, stream=side),
                    capi.group_norm(frames, 32, stream=side)))
        size = capi.linear_workspace(m, 640, 2560, capi.DTYPE_F32, capi.DTYPE_F32)
        torch.empty(max(size, 512), dtype=torch.uint8, device="cuda").fill_(255)
        torch.empty_like(want[0]).fill_(float("nan"))
    torch.cuda.synchronize()
    for y, z in got:
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])


def test_two_streams_at_once():
    """Calls of one shape on two streams, each with a workspace of its own."""
    import torch
    cases = [_operands(77, 5120, 512, PAIRS[1], "bfloat16", seed=s) for s in range(2)]
    want = [capi.linear(x, w, b, residual=r) for x, w, b, r in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, w, b, r) in enumerate(cases):
            got[i].append(capi.linear(x, w, b, residual=r, stream=streams[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


# few rows, tiles, the short k's kernel, no workspace
@pytest.mark.parametrize("m,k,n,workspace", [(1, 640, 96, True), (20, 133, 200, True), (300, 512, 264, True),
                                             (2500, 132, 2564, True), (2500, 64, 2564, True),
                                             (300, 512, 264, False)])
@pytest.mark.parametrize("y_type", Y_TYPES)
def test_fp32_rows_keep_their_bits(m, k, n, workspace, y_type):
    """Differences of two of a row's values, both near a thousand: exact products whose
    leading bits cancel.  A value is a sum of three bf16 terms at most, so a result is one
    of six products, added in five steps that are off by a step of fp32 (2 U) of the
    largest partial sum each, |a| + |b|; then it is rounded to y."""
    import torch
    import row_operators as ro
    draw = _gen(m + k + n)
    x = 1000.0 + draw(m, k)
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    a = torch.arange(n, device="cuda") % k
    b = (a + 1 + torch.arange(n, device="cuda") // k) % k
    rows = torch.arange(n, device="cuda")
    w[rows, a], w[rows, b] = 1.0, -1.0
    room = None if workspace else torch.empty(0, dtype=torch.uint8, device="cuda")
    got = capi.linear(x, w, out_dtype=getattr(torch, y_type), workspace=room)
    offs = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    parts = capi.grouped_linear(x, offs, torch.stack([w, w]), out_dtype=got.dtype, workspace=room)
    xd = x.double()
    want = xd[:, a] - xd[:, b]
    err = 5 * 2 * ro.U * (xd[:, a].abs() + xd[:, b].abs())
    for y in (got, parts):
        ro.check(y, want, err + ro.rounding(want.abs() + err, y.dtype))


@pytest.mark.parametrize("act", ["gelu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("y_type", Y_TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 96), (300, 64, 96), (77, 5120, 96), (2500, 32, 2564)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_activations_of_infinities(act, y_type, m, k, n, pair):
    """By a bias: +inf stays, a NaN too, -inf is -inf times 0, NaN as the formulas have
    it; on few rows, tiles, ranges of k and the short k's kernel, ragged rows among them."""
    import torch
    import row_operators as ro
    x, w, _, _ = _operands(m, k, n, pair, y_type)
    bias = torch.zeros(n, device="cuda")
    bias[::3] = float("inf")
    bias[1::6] = float("-inf")
    bias[4::6] = float("nan")
    for width in (n, n - 3):
        for y in (capi.linear(x, w[:width], bias[:width], ro.ACTS[act], out_dtype=getattr(torch, y_type)),
                  capi.grouped_linear(x, torch.tensor([0, m], dtype=torch.int32, device="cuda"),
                                      w[None, :width], bias[None, :width], ro.ACTS[act],
                                      out_dtype=getattr(torch, y_type))):
            assert (y[:, ::3] == float("inf")).all()
            assert y[:, 1::3].isnan().all()
            assert y[:, 2::3].isfinite().all()


@pytest.mark.parametrize("m,k,width", [(1, 64, 4001), (40, 64, 4000), (300, 64, 4001), (77, 5120, 4000),
                                       (2500, 32, 4001)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("workspace", [True, False])
def test_erf_gelu_of_fp32_results(m, k, width, pair, workspace):
    """To fp32's precision relative to the value, out into the negative tail; the
    values come by the bias, and with a residual."""
    import torch
    import row_operators as ro
    x, w, _, res = _operands(m, k, width, pair, "float32")
    x.zero_()
    bias = torch.linspace(-12, 12, width, device="cuda")
    v = bias.double().expand(m, width)
    room = None if workspace else torch.empty(0, dtype=torch.uint8, device="cuda")
    offs = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    for r in (None, res * 1e-6):
        want, err = ro.exact_gelu(v), ro.exact_gelu_error(v)
        if r is not None:
            want = want + r.double()
            err = err + ro.U * (want.abs() + err)
        ro.check(capi.linear(x, w, bias, capi.ACT_GELU, r, out_dtype=torch.float32, workspace=room), want, err)
        ro.check(capi.grouped_linear(x, offs, w[None], bias[None], capi.ACT_GELU, r, out_dtype=torch.float32,
                                     workspace=room), want, err)


@pytest.mark.parametrize("pair", PAIRS[1:], ids="-".join)
@pytest.mark.parametrize("m,k,n", [(40, 512, 96), (300, 320, 136), (1000, 2560, 2001)], ids=str)
def test_room_for_rows_that_the_tiles_cannot_read(m, k, n, pair, monkeypatch):
    """Rows of x apart by no multiple of eight elements, rows and weights that start at no
    16-byte boundary: the bindings' workspace has room to repack them, and the call takes
    the same kernels as with any amount."""
    import torch
    taken = []
    made = capi._workspace
    monkeypatch.setattr(capi, "_workspace", lambda w, s, x, size: (taken.append(size), made(w, s, x, size))[1])
    x, w, bias, res = _operands(m, k, n, pair, pair[0])
    offs = torch.tensor([0, m // 3, m], dtype=torch.int32, device="cuda")
    wg, bg = torch.stack([w, w]), torch.stack([bias, bias])
    for first, pad, odd in ((0, 4, 0), (3, 5, 0), (0, 0, 1), (4, 4, 4)):
        xw = torch.full((m, k + pad), float("nan"), dtype=x.dtype, device="cuda")
        xw = torch.cat([xw.flatten(), xw.new_zeros(first)])[first:first + m * (k + pad)].view(m, k + pad)[:, :k]
        xw.copy_(x)

        def moved(t):
            flat = torch.empty(t.numel() + odd, dtype=t.dtype, device="cuda")
            return flat[odd:].view_as(t).copy_(t)

        need = 2 * m * k + (2 * n * k if odd else 0)
        got = capi.linear(xw, moved(w), bias, capi.ACT_SILU, res)
        assert taken[-1] >= need
        _check(got, x, w, bias, "silu", res)
        plenty = torch.empty(8 * (need + 64 * m * n), dtype=torch.uint8, device="cuda")
        assert torch.equal(got, capi.linear(xw, moved(w), bias, capi.ACT_SILU, res, workspace=plenty))
        got = capi.grouped_linear(xw, offs, moved(wg), bg, capi.ACT_SILU, res)
        if m // 2 > 32:
            assert taken[-2] >= need
        _check(got, x, w, bias, "silu", res)


def test_fp32_rows_far_apart():
    """As test_rows_far_apart for fp32 rows: 70 of x, the residual and y over 9.4 GB each,
    and rows enough for the short k's kernel whose x is apart by less and by more than
    its offsets reach."""
    import torch
    m, k, n, far = 70, 72, 40, 2 ** 25 + 8
    x, w, bias, res = _operands(m, k, n, PAIRS[0], "float32")
    spread = [torch.empty(m * far, device="cuda") for _ in range(3)]
    xw, rw, yw = (t.as_strided((m, c), (far, 1)) for t, c in zip(spread, (k, n, n)))
    xw.copy_(x)
    rw.copy_(res)
    for args in ((xw, res, None), (x, res, yw), (x, rw, None), (xw, rw, rw)):
        got = capi.linear(args[0], w, bias, capi.ACT_SILU, args[1], out=args[2])
        _check(got, x, w, bias, "silu", res)
    del spread, xw, rw, yw
    m, k, n = 600, 60, 11000
    x, w, bias, _ = _operands(m, k, n, PAIRS[0], "bfloat16")
    for far in (2 ** 24 - 4, 2 ** 24 + 4):
        xw = torch.empty(m * far, device="cuda").as_strided((m, k), (far, 1))
        xw.copy_(x)
        _check(capi.linear(xw, w, bias, out_dtype=torch.bfloat16), x, w, bias, "none", None)
        del xw
    torch.cuda.empty_cache()
