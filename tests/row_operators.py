"""float64 forms of group norm, linear and grouped linear, and how far an fp32
computation of them may be off."""
import torch

from seedvr2_ncnn_amd import capi

U = 2.0 ** -24   # half a step of fp32, relative
ACTS = {"none": capi.ACT_NONE, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU,
        "gelu_tanh": capi.ACT_GELU_TANH}


def activation(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(1.5957691216057308 * (v + 0.044715 * v ** 3))
    return v


def activation_error(v, act):
    """Of the fp32 activation at v (its argument exact).  The exponentials'
    arguments z are off by 4 U |z| at most, which moves the result by as much
    relative to itself; their exponential, sum, reciprocal and product by 12 U.
    erfc's formula is off by 1.5e-7, times |v| / 2, and by 16 U."""
    y = activation(v, act).abs()
    if act == "silu":
        return (12 + 4 * v.abs()) * U * y
    if act == "gelu_tanh":
        return (12 + 4 * 1.6 * (v.abs() + 0.045 * v.abs() ** 3)) * U * y
    if act == "gelu":
        return (0.75e-7 + 16 * U) * v.abs()
    return torch.zeros_like(v)


def exact_gelu(v):
    return 0.5 * v * torch.erfc(-v / 2.0 ** 0.5)


def exact_gelu_error(v):
    """Of an erf-GELU as the product of v / 2 and erfc(-v / sqrt 2) in fp32: erfc's
    argument z is off by 2 U |z|, which moves it by no more than 2 z^2 + 1 times as much
    relative to itself (its slope is under 2 z + 1 times it); it is off by 4 steps (8 U),
    the products by 3 U, all relative to the value."""
    return (12 + 2 * (v * v + 1)) * U * exact_gelu(v).abs() + torch.finfo(torch.float32).tiny


def rounding(y, dtype):
    """Half a step of dtype at y; subnormals' step is the smallest number's."""
    info = torch.finfo(dtype)
    return y.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def finish(v, v_err, act, residual, dtype):
    """(result, bound) of residual + act(v) rounded to dtype, v off by v_err;
    the activations' slopes stay under 1.13 in magnitude."""
    y = activation(v, act)
    err = (1.13 if act != "none" else 1.0) * v_err + activation_error(v, act)
    if residual is not None:
        y = y + residual.double()
        err = err + U * y.abs()
    return y, err + rounding(y.abs() + err, dtype)


def linear(x, w, bias, act, residual, dtype):
    """k products summed in any order in fp32: (k + 2) U of the sum of their
    magnitudes, the bias one sum more; an fp32 x as two terms (16-bit results)
    is off by 2^-15 of itself."""
    xd, wt = x.double(), w.double().t().contiguous()
    v = xd @ wt
    size = xd.abs() @ wt.abs()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    err = (x.shape[1] + 3) * U * size
    if x.dtype == torch.float32 and dtype != torch.float32:
        err = err + 2.0 ** -15 * size
    return finish(v, err, act, residual, dtype)


def group_norm(x, groups, gamma, beta, eps, act, dtype):
    """Means and sums of squares are of deviations from a value of the group, at most
    `far`, the group's range, each.  A value passes through at most `steps` additions
    in a row: those of its thread (`length`, or 64 where a thread holds them all), of
    the parts of its workgroup that a lane adds (64 at most), of lanes (8) and of
    chunks (32 of a lane in these shapes).  So the mean is off by steps U far and,
    stored in fp32 three times, by 3 U of itself; the mean square by 2 steps U far^2
    and by what the parts' means are off, 2 mean_err far + mean_err^2."""
    f, p, c = x.shape
    xd = x.double().reshape(f, p, groups, c // groups)
    mean = xd.mean(dim=(1, 3), keepdim=True)
    d = xd - mean
    var = (d * d).mean(dim=(1, 3), keepdim=True)
    far = xd.amax(dim=(1, 3), keepdim=True) - xd.amin(dim=(1, 3), keepdim=True)
    length = min(max(16384 // c, -(-p // max(1, 1024 // f)), 1), p)
    steps = length + 64 + 64 + 8 + 32
    mean_err = steps * U * far + 3 * U * mean.abs()
    var_err = 2 * steps * U * far ** 2 + 2 * mean_err * far + mean_err ** 2
    std = (var + eps).sqrt()
    hat = d / std
    hat_err = (mean_err + 2 * U * d.abs()) / std + hat.abs() * (0.5 * var_err / (var + eps) + 4 * U)
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    v = hat.reshape(f, p, c) * g + b
    v_err = hat_err.expand_as(hat).reshape(f, p, c) * abs(g) + 2 * U * v.abs()
    return finish(v, v_err, act, None, dtype)


def group_norm_by_variance(x, groups, gamma, beta, eps, act, dtype):
    """As group_norm, for any distribution: what the statistics may be off by goes by a
    group's deviation alone, however far single values lie.

    A thread sums eight pixels about the first of them, K, then joins their mean b and
    sum of squared deviations M to those of the pixels before.  About K the squares sum
    to at most 9 M, (K - b)^2 being at most M: with eleven roundings of each and eight of
    their sum's, b's part off by 16 and 2, M is off by at most 29 * 9 U M = 261 U M.  The
    joining's difference of means is off by U times itself and 10.5 U sqrt(M), which moves
    its square, weighed by at most 8, by 14 U of itself and 84 U M.  Those sums are kept in
    two floats.  After that every sum is of squares or of deviations from a mean that
    is already near: 64 + 8 + 32 additions in a row at most, 54 where a thread holds its
    values, and 16 among channels; of means stored in fp32, 4 U of themselves.  So the
    variance is off by less than 600 U of itself, the mean by 200 U deviations."""
    f, p, c = x.shape
    xd = x.double().reshape(f, p, groups, c // groups)
    mean = xd.mean(dim=(1, 3), keepdim=True)
    d = xd - mean
    var = (d * d).mean(dim=(1, 3), keepdim=True)
    std = (var + eps).sqrt()
    mean_err = 200 * U * var.sqrt() + 4 * U * mean.abs()
    var_err = 600 * U * var + 2 * mean_err * var.sqrt() + mean_err ** 2
    hat = d / std
    hat_err = (mean_err + 2 * U * d.abs()) / std + hat.abs() * (0.5 * var_err / (var + eps) + 4 * U)
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    v = hat.reshape(f, p, c) * g + b
    v_err = hat_err.reshape(f, p, c) * abs(g) + 2 * U * v.abs()
    return finish(v, v_err, act, None, dtype)

def check(got, want, bound):
    off = (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"
