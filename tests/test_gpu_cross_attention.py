"""Cross attention against float64."""
import pytest
import torch

import mx_cross as mc
import row_operators as ro
from seedvr2_ncnn_amd import capi

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _sample(q, k, v, scale, kept, out_dtype):
    """All heads of one sample: (result, bound) [queries, heads, d]."""
    each = q.shape[1] // k.shape[1]
    pairs = [mc.attention(q[:, h], k[:, h // each], v[:, h // each], scale, kept, out_dtype)
             for h in range(q.shape[1])]
    return torch.stack([p[0] for p in pairs], 1), torch.stack([p[1] for p in pairs], 1)


def _padded(batch, lq, lk, heads, kv_heads, d, dtype, lengths=None, mask=None, out_dtype=None, scale=None,
            seed=0, poison=False, order="bshd", **kwargs):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def operand(n, h):
        t = _normal(gen, batch, n, h, d).to(dtype)
        if order == "bhsd":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if order == "sbhd":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        return t

    q, k, v = operand(lq, heads), operand(lk, kv_heads), operand(lk, kv_heads)
    kept = torch.ones(batch, lk, dtype=torch.bool, device="cuda")
    if lengths is not None:
        kept &= torch.arange(lk, device="cuda") < torch.tensor(lengths, device="cuda")[:, None]
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if mask is not None:
        kept &= mask
    if poison:
        k[~kept], v[~kept] = float("nan"), float("inf")
    got = capi.cross_attention(q, k, v, scale=scale, key_lengths=lengths, key_mask=mask, out_dtype=out_dtype,
                               **kwargs)
    assert got.dtype == (out_dtype or dtype)
    for b in range(batch):
        want, bound = _sample(q[b], k[b], v[b], d ** -0.5 if scale is None else scale, kept[b], got.dtype)
        ro.check(got[b], want, bound)
        if not kept[b].any():
            assert (got[b] == 0).all()
    return q, k, v, got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("batch,lq,lk,heads,kv_heads,d", [
    (1, 1, 1, 1, 1, 8), (1, 1, 1000, 4, 4, 128), (2, 3, 5, 2, 1, 64), (1, 33, 31, 3, 3, 40),
    (2, 129, 77, 4, 2, 128), (1, 257, 300, 2, 2, 64), (1, 64, 33, 8, 8, 72), (3, 100, 512, 5, 1, 96),
    (1, 130, 65, 2, 2, 256), (1, 70, 200, 2, 1, 136), (1, 500, 1, 2, 2, 64), (5, 1, 333, 20, 4, 128),
    (2, 7, 1500, 8, 1, 64), (1, 1, 5000, 16, 1, 128), (1, 2, 129, 3, 3, 256), (2, 2000, 16, 2, 2, 24),
    (1, 17, 2049, 1, 1, 120)])
def test_lengths(dtype, batch, lq, lk, heads, kv_heads, d):
    _padded(batch, lq, lk, heads, kv_heads, d, dtype, seed=lq + lk)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [1, 5, 40, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_key_lengths_and_masks_with_nan_behind_them(dtype, lq, d):
    lengths = [0, 1, 31, 32, 33, 64, 100, 199]
    _padded(8, lq, 199, 4, 2, d, dtype, lengths=lengths, poison=True)
    gen = torch.Generator(device="cuda").manual_seed(7)
    mask = torch.rand(8, 199, generator=gen, device="cuda") < 0.5
    mask[2] = False
    mask[3] = False
    mask[3, 198] = True
    mask[4, :150] = False
    mask[5, 64:] = False
    mask[6] = torch.arange(199, device="cuda") % 64 == 63
    _padded(8, lq, 199, 4, 2, d, dtype, mask=mask, poison=True)
    _padded(8, lq, 199, 4, 4, d, dtype, mask=mask, lengths=lengths[::-1], poison=True)
    _padded(8, lq, 199, 2, 2, d, dtype, mask=mask[:, :199], lengths=[199] * 8, poison=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_long_masked_keys_of_few_queries(dtype):
    """Ranges of keys that the mask leaves empty."""
    mask = torch.zeros(3, 4000, dtype=torch.bool, device="cuda")
    mask[0, 3999] = True
    mask[1, 17] = True
    _padded(3, 2, 4000, 4, 1, 128, dtype, mask=mask, poison=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strided_operands(dtype):
    for order in ("bhsd", "sbhd"):
        _padded(3, 70, 90, 4, 2, 64, dtype, order=order)
        _padded(3, 1, 900, 4, 2, 64, dtype, order=order)
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = _normal(gen, 2, 100, 12, 64).to(dtype)   # a fused projection's q, k, v
    q, k, v = wide[:, :, :4], wide[:, :, 4:8], wide[:, :, 8:]
    out = torch.full((2, 100, 5, 67), 9.0, dtype=dtype, device="cuda")
    got = capi.cross_attention(q, k, v, out=out[:, :, :4, 1:65])
    assert (out[:, :, 4] == 9).all() and (out[..., 0] == 9).all() and (out[..., 65:] == 9).all()
    for b in range(2):
        ro.check(got[b], *_sample(q[b], k[b], v[b], 64 ** -0.5, None, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [1, 90])
def test_broadcast_keys(dtype, lq):
    """One prompt for every sample, one head for all: strides of zero."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = _normal(gen, 3, lq, 4, 64).to(dtype)
    k, v = (_normal(gen, 1, 50, 1, 64).to(dtype).expand(3, 50, 4, 64) for _ in range(2))
    got = capi.cross_attention(q, k, v)
    for b in range(3):
        ro.check(got[b], *_sample(q[b], k[b], v[b], 64 ** -0.5, None, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [1, 90])
def test_one_mask_for_all_samples(dtype, lq):
    mask = torch.arange(70, device="cuda") % 3 != 0
    _padded(4, lq, 70, 4, 2, 64, dtype, mask=mask.expand(4, 70), poison=True)
    wide = torch.zeros(4, 100, dtype=torch.uint8, device="cuda")
    wide[:, 5:75] = mask * 7   # any byte but nought
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (_normal(gen, 4, n, 2, 64).to(dtype) for n in (lq, 70, 70))
    a = capi.cross_attention(q, k, v, key_mask=wide[:, 5:75])
    assert torch.equal(a, capi.cross_attention(q, k, v, key_mask=mask.expand(4, 70)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 104, 256])
@pytest.mark.parametrize("lq", [3, 700])
@pytest.mark.parametrize("kept", [(0, 40), (999, 1000), (96, 128), (200, 900)])
def test_whole_tiles_left_out(dtype, d, lq, kept):
    keys = torch.arange(1000, device="cuda")
    mask = (keys >= kept[0]) & (keys < kept[1])
    both = torch.stack([mask, keys % 300 == 5])
    _padded(2, lq, 1000, 2, 1, d, dtype, mask=both, poison=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_calls_side_by_side(dtype):
    """Two streams at once, each call with a workspace of its own."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    sets = [tuple(_normal(gen, 1, n, 4, 128).to(dtype) for n in (lq, 4000, 4000)) for lq in (1, 200)]
    want = [capi.cross_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(sets):
            got[i].append(capi.cross_attention(*s, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_far_rows_of_keys(dtype):
    """Key rows so far apart that a tile's reach passes 32 bits from the first one."""
    n, step = 70, 1 << 23
    flat = torch.empty((n - 1) * step + 64, dtype=dtype, device="cuda")
    k = flat.as_strided((1, n, 1, 64), (0, step, 64, 1))
    gen = torch.Generator(device="cuda").manual_seed(12)
    k.copy_(_normal(gen, 1, n, 1, 64))
    q, v = _normal(gen, 1, 40, 1, 64).to(dtype), _normal(gen, 1, n, 1, 64).to(dtype)
    for lq in (1, 40):
        got = capi.cross_attention(q[:, :lq], k, v)
        ro.check(got[0], *_sample(q[0, :lq], k[0], v[0], 64 ** -0.5, None, dtype))


@pytest.mark.parametrize("batch,heads", [(1 << 20, 20), ((1 << 24) + 2, 1)])
def test_more_tiles_than_a_launch_has(batch, heads):
    """A key a sample: out is v, to the bit, and nought where the key is masked."""
    v = torch.arange(batch * heads * 8, device="cuda").remainder_(253).bfloat16().view(batch, 1, heads, 8)
    lengths = (torch.arange(batch, device="cuda") % 7 != 0).int()
    mask = torch.arange(batch, device="cuda").view(batch, 1) % 5 != 0
    got = capi.cross_attention(v, v, v, key_lengths=lengths, key_mask=mask)
    v[(lengths == 0) | ~mask[:, 0]] = 0
    assert torch.equal(got, v)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("out_dtype", TYPES, ids=str)
def test_out_types_and_scales(dtype, out_dtype):
    for lq in (2, 150):
        _padded(1, lq, 100, 2, 2, 64, dtype, out_dtype=out_dtype, scale=0.3)
        _padded(1, lq, 100, 2, 2, 128, dtype, out_dtype=out_dtype, scale=-0.05)
        _padded(1, lq, 100, 2, 2, 64, dtype, out_dtype=out_dtype, scale=0.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [1, 200])
@pytest.mark.parametrize("size", [8.0, 60.0])
def test_large_scores(dtype, lq, size):
    """Weights that all but vanish, rising and falling maxima along the keys."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = _normal(gen, 1, lq, 2, 64), _normal(gen, 1, 700, 2, 64), _normal(gen, 1, 700, 2, 64)
    q *= size
    k[:, :350] *= torch.linspace(0.1, 2.0, 350, device="cuda")[:, None, None]
    k[:, 350:] *= torch.linspace(2.0, 0.1, 350, device="cuda")[:, None, None]
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    got = capi.cross_attention(q, k, v)
    want, bound = _sample(q[0], k[0], v[0], 64 ** -0.5, None, dtype)
    ro.check(got[0], want, bound)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [3, 140])
def test_infinite_scores(dtype, lq):
    """-inf among the scores is a weight of nought; NaN makes its row NaN."""
    q = torch.zeros(1, lq, 1, 64, dtype=dtype, device="cuda")
    q[0, 0, 0, 0], q[0, 1, 0, 0], q[0, 2, 0, 1] = 1.0, -1.0, 1.0
    k = torch.zeros(1, 40, 1, 64, dtype=dtype, device="cuda")
    k[0, ::2, 0, 0] = -float("inf")
    v = torch.arange(40, device="cuda").to(dtype)[None, :, None, None].expand(1, 40, 1, 64).contiguous()
    got = capi.cross_attention(q, k, v)[0, :, 0].float()
    assert got[1:].isnan().all()   # 0 * inf
    k = torch.full((1, 40, 1, 64), -float("inf"), dtype=dtype, device="cuda")
    k[0, 1::2] = 0.0
    got = capi.cross_attention(torch.ones_like(q), k, v)[0, :, 0].float()
    # the mean of the odd ones; 20 weights of one and their sum are exact
    assert (got == 20.0).all()


def _ragged(queries, keys, heads, kv_heads, d, dtype, spare=3, mask=None, seed=0, **kwargs):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    nq, nk = sum(queries), sum(keys)
    q = _normal(gen, nq + spare, heads, d).to(dtype)
    kv = _normal(gen, nk + spare, 2 * kv_heads, d).to(dtype)
    k, v = kv[:, :kv_heads], kv[:, kv_heads:]
    k[nk:] = float("nan")
    ends = [[0], [0]]
    for e, sizes in zip(ends, (queries, keys)):
        for s in sizes:
            e.append(e[-1] + s)
    qo, ko = (torch.tensor(e, dtype=torch.int32, device="cuda") for e in ends)
    out = torch.full((nq + spare, heads, d), 5.0, dtype=dtype, device="cuda")
    if mask is not None:
        k[~mask], v[~mask] = float("inf"), float("nan")
    assert capi.cross_attention(q, k, v, q_offsets=qo, k_offsets=ko, key_mask=mask, out=out, **kwargs) is out
    assert (out[nq:] == 5).all()
    for b in range(len(queries)):
        qs, ks = slice(ends[0][b], ends[0][b + 1]), slice(ends[1][b], ends[1][b + 1])
        if queries[b]:
            ro.check(out[qs], *_sample(q[qs], k[ks], v[ks], d ** -0.5, None if mask is None else mask[ks], dtype))
            if keys[b] == 0:
                assert (out[qs] == 0).all()
    return q, k, v, qo, ko, out


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries,keys,heads,kv_heads,d", [
    ([1], [1], 1, 1, 64), ([5, 0, 130, 1], [77, 3, 0, 40], 4, 2, 128), ([300, 20, 7], [10, 200, 33], 2, 2, 64),
    ([1] * 40, list(range(0, 120, 3)), 8, 2, 128), ([3] * 70, [9] * 70, 2, 1, 40), ([0, 0, 2], [0, 5, 900], 4, 4, 64),
    ([1, 1, 1, 1], [3000, 10, 0, 900], 5, 1, 128)])
def test_ragged(dtype, queries, keys, heads, kv_heads, d):
    _ragged(queries, keys, heads, kv_heads, d, dtype)
    gen = torch.Generator(device="cuda").manual_seed(4)
    mask = torch.rand(sum(keys) + 3, generator=gen, device="cuda") < 0.6
    mask[sum(keys):] = False
    _ragged(queries, keys, heads, kv_heads, d, dtype, mask=mask)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_many_queries_on_few_keys(dtype):
    _padded(1, 14000, 77, 20, 20, 128, dtype)
    _padded(2, 9001, 128, 16, 8, 72, dtype, lengths=[128, 0], poison=True)
    mask = torch.rand(3, 97, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") < 0.7
    mask[1] = False
    mask[2, :40] = False
    _padded(3, 6000, 97, 16, 16, 128, dtype, mask=mask, poison=True)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_many_queries_on_few_keys_but_for_some_samples(dtype):
    """Samples of more keys than others have on average, by far."""
    queries, keys = [9000, 1, 5000, 130, 0, 700], [20, 300, 129, 0, 9, 128]
    _ragged(queries, keys, 20, 20, 128, dtype)
    mask = torch.rand(sum(keys) + 3, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") < 0.5
    mask[sum(keys):] = False
    _ragged(queries, keys, 20, 20, 128, dtype, mask=mask)


def test_offsets_outside_the_rows_are_taken_as_their_ends():
    q, k = torch.randn(20, 2, 64, device="cuda"), torch.randn(30, 2, 64, device="cuda")
    v = torch.randn(30, 2, 64, device="cuda")
    far = torch.tensor([-5, 10, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    near_q = torch.tensor([0, 10, 20], dtype=torch.int32, device="cuda")
    near_k = torch.tensor([0, 10, 30], dtype=torch.int32, device="cuda")
    for t in (torch.float32, torch.bfloat16):
        a = capi.cross_attention(q.to(t), k.to(t), v.to(t), q_offsets=far, k_offsets=far)
        b = capi.cross_attention(q.to(t), k.to(t), v.to(t), q_offsets=near_q, k_offsets=near_k)
        assert torch.equal(a, b)
    lengths = torch.tensor([99, -3], dtype=torch.int32, device="cuda")
    y = capi.cross_attention(q.view(2, 10, 2, 64), k.view(2, 15, 2, 64), v.view(2, 15, 2, 64), key_lengths=lengths)
    assert torch.equal(y[:1], capi.cross_attention(q.view(2, 10, 2, 64)[:1], k.view(2, 15, 2, 64)[:1],
                                                   v.view(2, 15, 2, 64)[:1]))
    assert (y[1] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_nothing_to_do(dtype):
    q = torch.randn(2, 3, 4, 64, device="cuda").to(dtype)
    k = torch.randn(2, 0, 2, 64, device="cuda").to(dtype)
    assert (capi.cross_attention(q, k, k) == 0).all()
    k = torch.randn(2, 5, 2, 64, device="cuda").to(dtype)
    assert capi.cross_attention(q[:, :0], k, k).shape == (2, 0, 4, 64)
    assert capi.cross_attention(q[:0], k[:0], k[:0]).shape == (0, 3, 4, 64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [1, 300])
def test_in_place_and_without_workspace(dtype, lq):
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = (_normal(gen, 2, n, 4, 64).to(dtype) for n in (lq, 3000, 3000))
    want = capi.cross_attention(q, k, v)
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    got = capi.cross_attention(q, k, v, workspace=none)
    for b in range(2):
        ro.check(got[b], *_sample(q[b], k[b], v[b], 64 ** -0.5, None, dtype))
    assert capi.cross_attention(q, k, v, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq,lk", [(1, 3000), (300, 100)])
def test_graphs_and_streams(dtype, lq, lk):
    """Two captured calls with workspaces of their own, replayed between eager work, the
    lengths changed in between; equal every time."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    sets = [tuple(_normal(gen, 2, n, 4, 64).to(dtype) for n in (lq, lk, lk)) for _ in range(2)]
    lengths = torch.tensor([lk, lk // 2], dtype=torch.int32, device="cuda")
    other = torch.tensor([7, lk], dtype=torch.int32, device="cuda")
    first = [capi.cross_attention(*s, key_lengths=lengths) for s in sets]
    second = [capi.cross_attention(*s, key_lengths=other) for s in sets]
    held = lengths.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = [torch.zeros_like(s[0]) for s in sets]
    graphs = []
    for s, o in zip(sets, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            capi.cross_attention(*s, key_lengths=held, out=o)
        graphs.append(g)
    for turn in range(4):
        held.copy_(other if turn % 2 else lengths)
        for g, o, w in zip(graphs, outs, second if turn % 2 else first):
            o.zero_()
            g.replay()
            assert torch.equal(capi.cross_attention(*sets[0], key_lengths=lengths), first[0])
            torch.cuda.synchronize()
            assert torch.equal(o, w)
    y = capi.cross_attention(*sets[1], key_lengths=lengths, stream=side)
    side.synchronize()
    assert torch.equal(y, first[1])


def test_text_sublayer():
    """A text-conditioned sublayer as it would be used: projections with weights in four bits,
    cross attention to the prompts' states, the out projection onto the residual stream; each
    step against float64 on its own inputs."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    tokens, text, width, heads, d = [400, 130], [77, 12], 256, 4, 64
    x, states = _normal(gen, sum(tokens), width), _normal(gen, sum(text), 192).bfloat16()

    def weight(n, k):
        w = _normal(gen, n, k) * k ** -0.5
        return capi.mx_quantize(w), mc.values(*mc.quantize(w), k).cuda()

    (wq, wqv), (wkv, wkvv), (wo, wov) = weight(width, width), weight(2 * width, 192), weight(width, width)
    xq = capi.mx_quantize(x)
    q = capi.mx_linear(xq, wq)
    kv = capi.mx_linear(states, wkv)
    ro.check(q, *mc.linear(capi.mx_dequantize(xq, torch.float32).double(), wqv, None, "none", None, torch.bfloat16))
    ro.check(kv, *mc.linear(states.double(), wkvv, None, "none", None, torch.bfloat16))
    qo = torch.tensor([0, 400, 530], dtype=torch.int32, device="cuda")
    ko = torch.tensor([0, 77, 89], dtype=torch.int32, device="cuda")
    q3, k3, v3 = q.view(-1, heads, d), kv[:, :width].view(-1, heads, d), kv[:, width:].view(-1, heads, d)
    o = capi.cross_attention(q3, k3, v3, q_offsets=qo, k_offsets=ko)
    for qs, ks in ((slice(0, 400), slice(0, 77)), (slice(400, 530), slice(77, 89))):
        ro.check(o[qs], *_sample(q3[qs], k3[ks], v3[ks], d ** -0.5, None, torch.bfloat16))
    oq = capi.mx_quantize(o.view(-1, width))
    y = capi.mx_linear(oq, wo, residual=x, out=x.clone())
    ro.check(y, *mc.linear(capi.mx_dequantize(oq, torch.float32).double(), wov, None, "none", x, torch.float32))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 3000), (200, 1), (200, 97), (14000, 77)])
@pytest.mark.parametrize("d", [64, 128])
def test_equal_scores_of_any_size(dtype, lq, lk, d):
    """Scores times log2 e of 2^20 to 2^36, in fp32 up to 2^120, of either sign: as the
    weights are equal, small numbers in v sum exactly and out is their mean, rounded in the
    division (U) and to its type."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    v = torch.randint(-8, 9, (1, lk, 1, d), generator=gen, device="cuda").to(dtype)
    mean = v.double().mean(dim=1, keepdim=True)
    bound = mean.abs() * 2 * ro.U
    bound = bound + ro.rounding(mean.abs() + bound, dtype)
    sizes = [(1 + j / 8) * 2.0 ** e for e in range(10, 16) for j in range(8) if dtype != torch.float16 or e < 15]
    if dtype == torch.float32:
        sizes += [1.125 * 2.0 ** e for e in (20, 30, 40, 58)]
    for i, size in enumerate(sizes):
        q = torch.full((1, lq, 1, d), size, device="cuda").to(dtype)
        k = torch.full((1, lk, 1, d), size, device="cuda").to(dtype)
        got = capi.cross_attention(q, -k if i % 3 == 2 else k, v, scale=-0.0884 if i % 3 == 1 else None)
        ro.check(got, mean.expand(1, lq, 1, d), bound)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq,lk", [(1, 3000), (3, 250), (200, 250), (14000, 77)])
@pytest.mark.parametrize("exponent", [12, 20, 24, 26, 28])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_far_scores_that_differ_by_steps(dtype, lq, lk, exponent, order):
    """Scores 2^exponent + i steps of fp32, i up to 127, whose products and sums are exact.  An
    exponential's argument, a difference of scores times a factor, is off by 3 U of itself, at
    most 32 here, the exponential by 4 U; each rescale of the sums by as much again and U.  Of
    weights, sums and division the rest, as in mx_cross.attention."""
    d = 64 if lq == 3 else 128
    big = 2.0 ** (exponent // 2)
    step = 2.0 ** (exponent - 23)
    i = torch.arange(lk, device="cuda") * 127 // max(lk - 1, 1)
    if order == "falling":
        i = i.flip(0)
    elif order == "mixed":
        i = i[torch.randperm(lk, generator=torch.Generator(device="cuda").manual_seed(15), device="cuda")]
    q = torch.zeros(1, lq, 1, d, device="cuda")
    k = torch.zeros(1, lk, 1, d, device="cuda")
    q[..., 3], k[..., 3] = big, 2.0 ** exponent / big
    q[..., 41], k[..., 41] = 2.0 ** (exponent // 2 - 12), (i * step / 2.0 ** (exponent // 2 - 12))[None, :, None]
    gen = torch.Generator(device="cuda").manual_seed(14)
    v = _normal(gen, 1, lk, 1, d).to(dtype)
    q, k = q.to(dtype), k.to(dtype)
    assert torch.equal((q[0, 0, 0].double() * k[0, :, 0].double()).sum(1), 2.0 ** exponent + i.double() * step)
    scale = 0.25 / step
    got = capi.cross_attention(q, k, v, scale=scale)
    w = torch.softmax(0.25 * i.double(), dim=0)
    want = w @ v[0, :, 0].double()
    tiles = (lk + 31) // 32
    rel = 2 * (3 * ro.U * 32 + 4 * ro.U + tiles * 5 * ro.U) + (2 * lk + 8) * ro.U
    if dtype != torch.float32:
        rel += torch.finfo(dtype).eps / 2
    bound = rel * (w @ v[0, :, 0].double().abs())
    if dtype == torch.float16:
        bound = bound + v[0, :, 0].double().abs().sum(dim=0) * 2.0 ** -25
    ro.check(got[0, :, 0], want.expand(lq, d), (bound + ro.rounding(want.abs() + bound, dtype)).expand(lq, d))


@pytest.mark.parametrize("lq", [1, 200])
@pytest.mark.parametrize("scale,size", [(0.0, 1e19), (1e-40, 1e19), (1e-38, 1.0), (-1e-45, 1e19), (3e38, 1e-20), (-3e38, 1e-15)])
def test_smallest_and_largest_scales(lq, scale, size):
    """Scores of 10^37 under a scale of nought or next to it weigh alike, within 2^-21 of the
    argument; so do equal ones under the largest."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    v = _normal(gen, 1, 300, 2, 64)
    q = torch.full((1, lq, 2, 64), size / 8, device="cuda")
    k = q[:, :1].expand(1, 300, 2, 64).clone()
    if abs(scale) < 1:
        k *= torch.where(torch.arange(300, device="cuda") % 2 == 0, 1.0, -1.0)[:, None, None]
    got = capi.cross_attention(q, k, v, scale=scale)
    want = v.double().mean(dim=1, keepdim=True).expand(1, lq, 2, 64)
    s = 64 * (size / 8) ** 2 * abs(scale) if abs(scale) < 1 else 0.0
    bound = (2 * (s + 2.0 ** -20) + 700 * ro.U) * v.double().abs().mean(dim=1, keepdim=True).expand_as(want)
    ro.check(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("batch", [63, 64, 65, 66, 1000, 4097])
def test_many_ragged_samples(dtype, batch):
    """Samples of no, one and several tiles, without keys and with, rows ahead of the first one
    and behind the last: each as a call of its own gives it, but for the order of a row's sums."""
    gen = torch.Generator().manual_seed(batch)
    nq = torch.randint(0, 4, (batch,), generator=gen) * torch.randint(0, 90, (batch,), generator=gen)
    nk = torch.randint(0, 3, (batch,), generator=gen) * torch.randint(0, 40, (batch,), generator=gen)
    nq[batch // 3:batch // 2] = 0
    nq[-1] = 300
    qo, ko = (torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]) + 7 for n in (nq, nk))
    q = torch.randn(int(qo[-1]) + 5, 4, 64, generator=gen).to(dtype).cuda()
    k, v = (torch.randn(int(ko[-1]) + 5, 2, 64, generator=gen).to(dtype).cuda() for _ in range(2))
    out = torch.full_like(q, 5.0)
    capi.cross_attention(q, k, v, q_offsets=qo.int().cuda(), k_offsets=ko.int().cuda(), out=out)
    assert (out[:7] == 5).all() and (out[int(qo[-1]):] == 5).all()
    longest = int(nk.max())
    sample = torch.repeat_interleave(torch.arange(batch), nq)   # of each row
    index = (ko[:-1, None] + torch.arange(longest)).clamp(max=int(ko[-1]))[sample].cuda()
    kept = (torch.arange(longest) < nk[:, None])[sample].cuda()
    rows = out[7:int(qo[-1])]
    for at in range(0, rows.shape[0], 20000):   # in 64 bits, all heads of a row at once
        qs = q[7 + at:7 + at + 20000][:len(rows) - at].double()[:, :, None]
        ks, vs = (t[index[at:at + 20000]].double().transpose(1, 2).repeat_interleave(2, 1) for t in (k, v))
        s = (qs * ks).sum(-1) * 0.125
        size = (qs.abs() * ks.abs()).sum(-1) * 0.125
        s = s.masked_fill(~kept[at:at + 20000, None], -float("inf"))
        some = kept[at:at + 20000].any(1)[:, None, None]
        w = torch.where(some, torch.softmax(s, -1), torch.zeros((), dtype=torch.float64, device="cuda"))
        want = (w[..., None] * vs).sum(2)
        # as in mx_cross.attention
        arg = 68 * ro.U * size.amax(-1) + 2 * ro.U * 1.45 * torch.where(w > 0, s, 0.0).abs().amax(-1)
        rel = 2 * (2 * arg + 4 * ro.U) + (2 * longest + 8) * ro.U
        rel = rel + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0)
        bound = (w[..., None] * vs.abs()).sum(2) * rel[..., None]
        if dtype == torch.float16:
            bound = bound + (kept[at:at + 20000, None, :, None] * vs.abs()).sum(2) * 2.0 ** -25
        ro.check(rows[at:at + 20000], want, bound + ro.rounding(want.abs() + bound, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads", [1, 6])
def test_a_million_ragged_samples(dtype, heads):
    """A key a sample: out is its v, to the bit; none: nought."""
    batch = (1 << 20) + 3
    number = torch.arange(batch, device="cuda")
    nq, nk = (number % 3).int(), (number % 5 != 0).int()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo, ko = (torch.cat([zero, n.cumsum(0).int()]) for n in (nq, nk))
    rows, keys = int(qo[-1]), int(ko[-1])
    q = torch.ones(rows, heads, 8, dtype=dtype, device="cuda")
    v = (number[:keys, None, None] * 7 + torch.arange(8 * heads, device="cuda").view(heads, 8)).remainder(251).to(dtype)
    sample = torch.repeat_interleave(number, nq)
    want = v[ko[sample].long().clamp(max=keys - 1)]
    want[nk[sample] == 0] = 0
    assert torch.equal(capi.cross_attention(q, v, v, q_offsets=qo, k_offsets=ko), want)


def test_offsets_in_disorder_stay_within_the_rows():
    """What descending offsets give is nobody's business, but rows that no sample can have keep
    their values, and the calls end."""
    gen = torch.Generator().manual_seed(21)
    for batch in (5, 64, 65, 700):
        qo = torch.randint(-50, 900, (batch + 1,), generator=gen, dtype=torch.int32).cuda()
        ko = torch.randint(-50, 900, (batch + 1,), generator=gen, dtype=torch.int32).cuda()
        q = torch.randn(1000, 2, 64, device="cuda")
        for t in (torch.float32, torch.bfloat16):
            out = torch.full((1000, 2, 64), 5.0, device="cuda", dtype=t)
            capi.cross_attention(q.to(t)[:800], q.to(t)[:800], q.to(t)[:800], q_offsets=qo, k_offsets=ko, out=out[:800])
            torch.cuda.synchronize()
            assert (out[800:] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_as_many_rows_as_there_may_be(dtype):
    """One kv head's 2^30 rows; query i of head j is that of i + 1 and j - 1, and so is its row."""
    lq, heads = 1 << 25, 32
    gen = torch.Generator(device="cuda").manual_seed(22)
    flat = _normal(gen, lq + heads, 8).to(dtype)
    q = flat.as_strided((1, lq, heads, 8), (0, 8, 8, 1))
    k, v = (_normal(gen, 1, 5, 1, 8).to(dtype) for _ in range(2))
    out = torch.full((1, lq, heads, 8), 9.0, dtype=torch.bfloat16, device="cuda")
    capi.cross_attention(q, k, v, out=out)
    assert torch.equal(out[0, 1:, :-1], out[0, :-1, 1:])
    for part in (slice(0, 3000), slice(lq - 3000, lq), slice(lq // 2 - 1500, lq // 2 + 1500)):
        ro.check(out[0, part], *_sample(q[0, part], k[0], v[0], 8 ** -0.5, None, torch.bfloat16))


@pytest.mark.parametrize("batch,heads", [((1 << 24) + 5, 1), ((1 << 22) + 1, 5)])
def test_more_ragged_tiles_than_a_launch_has(batch, heads):
    """A query and a key a sample: out is v, to the bit."""
    v = torch.arange(batch * heads * 8, device="cuda").remainder_(253).bfloat16().view(batch, heads, 8)
    offsets = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    assert torch.equal(capi.cross_attention(v, v, v, q_offsets=offsets, k_offsets=offsets), v)


def test_more_tiles_than_32_bits_count():
    """2^31 samples and heads of one row on one key: out is v, to the bit."""
    batch, heads = 1 << 30, 2
    flat = torch.arange(8 * (batch + heads), dtype=torch.int32, device="cuda").remainder_(253).bfloat16()
    v = flat.as_strided((batch, 1, heads, 8), (8, 8, 8, 1))
    out = torch.full((batch, 1, heads, 8), 9.0, dtype=torch.bfloat16, device="cuda")
    capi.cross_attention(v, v, v, out=out)
    for h in range(heads):
        assert torch.equal(out[:, 0, h], flat.view(-1, 8)[h:h + batch])


def _block_mask(batch, lk):
    """Masks of more than one block of bits: kept keys at the blocks' borders, half of all, one
    far from the end, whole blocks left out."""
    keys = torch.arange(lk, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(lk)
    mask = torch.rand(batch, lk, generator=gen, device="cuda") < 0.5
    near = keys.remainder(8192)
    mask[1] = (near < 2) | (near > 8189) | (keys >= lk - 2)
    if batch > 2:
        mask[2] = keys == 8200
    if batch > 3:
        mask[3] = (keys < 40) | ((keys >= 8192) & (keys % 5 == 0) & (keys < 16384))
    return mask


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lk", [8191, 8192, 8193, 8225, 16384, 16385, 20000])
@pytest.mark.parametrize("lq,d", [(1, 128), (40, 64), (70, 136)])
def test_masks_of_several_blocks(dtype, lk, lq, d):
    """Ranges of keys that begin and end inside blocks, waves without rows, NaN behind the mask."""
    _padded(4, lq, lk, 2, 1, d, dtype, mask=_block_mask(4, lk), poison=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lk", [8193, 16385, 25000])
def test_masks_of_several_blocks_in_one_range(dtype, lk):
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    _padded(2, 300, lk, 2, 2, 64, dtype, mask=_block_mask(2, lk), poison=True, workspace=none)
    _padded(2, 20, lk, 2, 2, 128, dtype, mask=_block_mask(2, lk), lengths=[lk - 3, lk // 2], poison=True,
            workspace=none)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_a_sample_of_several_blocks_among_short_ones(dtype):
    """The kernel that keeps short samples' keys, read again for every 128 rows of a long one."""
    queries, keys = [9000, 300, 700] + [1500] * 157, [20, 17000, 9] + [20] * 157
    mask = torch.rand(sum(keys) + 3, generator=torch.Generator(device="cuda").manual_seed(23), device="cuda") < 0.5
    mask[sum(keys):] = False
    mask[20 + 8192:20 + 8200] = False
    _ragged(queries, keys, 4, 4, 128, dtype, mask=mask)
