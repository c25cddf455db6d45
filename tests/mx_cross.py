"""float64 forms of MXFP4 quantisation and products and of cross attention, and how far a
computation of them in fp32 may be off."""
import torch

from row_operators import U, finish, rounding

NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def blocks(k):
    return (k + 31) // 32


def quantize(x):
    """(codes [m, 32 blocks] of 0..15, scale bytes [m, blocks]) of rows x on the CPU."""
    m, k = x.shape
    full = torch.zeros(m, blocks(k) * 32, dtype=torch.float64)
    full[:, :k] = x.double().cpu()
    full = full.view(m, -1, 32)
    bad = ~torch.isfinite(full).all(dim=2)
    high = torch.where(bad[:, :, None], torch.zeros((), dtype=torch.float64), full).abs().amax(dim=2)
    exponent = (torch.frexp(high)[1] - 3).clamp(min=-127)
    exponent[high == 0] = -127
    v = torch.ldexp(torch.where(bad[:, :, None], torch.zeros((), dtype=torch.float64), full),
                    -exponent[:, :, None])
    grid = torch.tensor(NUMBERS, dtype=torch.float64)
    near = (v.abs()[..., None] - grid).abs()
    low = near.argmin(dim=-1)   # the lower of two as near
    tie = torch.gather(near, -1, (low + 1).clamp(max=7)[..., None])[..., 0] == near.min(dim=-1).values
    code = torch.where(tie & (low % 2 == 1) & (low < 7), low + 1, low)
    code = code + 8 * torch.signbit(full).long()
    code[bad] = 0
    scale = exponent + 127
    scale[bad] = 255
    return code.view(m, -1), scale


def pack(code, scale, device="cuda", stride=None):
    """MxRows' codes and scales, scale rows `stride` apart (None: a multiple of 16)."""
    m, b = scale.shape
    c = code.to(torch.uint8).view(m, b * 16, 2)
    stride = (b + 15) // 16 * 16 if stride is None else stride
    s = torch.full((m, stride), 255, dtype=torch.uint8)   # NaNs between the rows
    s[:, :b] = scale.to(torch.uint8)
    return (c[:, :, 0] | (c[:, :, 1] << 4)).contiguous().to(device), s.to(device)[:, :b]


def unpack(codes):
    c = codes.cpu().long()
    return torch.stack([c & 15, c >> 4], dim=2).flatten(1)


def values(code, scale, k):
    grid = torch.tensor(NUMBERS, dtype=torch.float64)
    v = grid[code & 7] * torch.where(code > 7, -1.0, 1.0).double()
    factor = torch.ldexp(torch.ones(scale.shape, dtype=torch.float64), scale.long() - 127)
    factor[scale == 255] = float("nan")
    return (v.view(scale.shape[0], -1, 32) * factor[:, :, None]).flatten(1)[:, :k]


def linear(x, w, bias, act, residual, dtype):
    """Exact products, k of them summed in fp32 in any order, the bias one sum more.  x, w:
    float64 values."""
    wt = w.t().contiguous()
    v = x @ wt
    size = x.abs() @ wt.abs()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    return finish(v, (x.shape[1] + 3) * U * size, act, residual, dtype)


def attention(q, k, v, scale, kept, out_dtype):
    """(result, bound) of one sample and head, q [queries, d], k and v [keys, d], kept: the
    keys' truth values or None.

    A score is d products summed in fp32 and two factors (scale, log2 e): off by
    (d + 4) U of the sum of their magnitudes.  The exponential's argument is off by that of
    the score and of the maximum, and by 2 U of both; the exponential by 4 U of itself.
    So a weight is off by twice the largest such error relative to itself, the sum of n
    weights by n U more, and their division by 4 U; products and sums with v by (n + 2) U.
    16-bit operands: a weight is rounded to their type, by half a step of itself, fp16's
    subnormal weights by 2^-25 of the largest."""
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    if kept is not None:
        k, v = k[kept], v[kept]
    n = k.shape[0]
    if n == 0:
        zero = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
        return zero, zero + 1e-300
    kt = k.t().contiguous()
    s = q @ kt * scale
    size = (q.abs() @ kt.abs()) * abs(scale)
    s_err = ((q.shape[1] + 4) * U * size).amax(dim=1, keepdim=True)
    arg = s_err + 2 * U * 1.45 * s.abs().amax(dim=1, keepdim=True)
    w = torch.softmax(s, dim=1)
    o = w @ v
    rel = 2 * (2 * arg + 4 * U) + (2 * n + 8) * U
    if dtype != torch.float32:
        rel = rel + torch.finfo(dtype).eps / 2
    err = (w @ v.abs()) * rel
    if dtype == torch.float16:
        err = err + v.abs().sum(dim=0, keepdim=True) * 2.0 ** -25
    return o, err + rounding(o.abs() + err, out_dtype)
