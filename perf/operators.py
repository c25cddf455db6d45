"""Group norm, linear and grouped linear as measurable cases.

Three operators that stand around the DiT's and the VAE's attention and
convolutions.  A case is a dict of plain values; "kind" names its operator:

  norm      group norm of channels-last frames, with an activation
            (capi.group_norm):  y = act((x - mean) / sqrt(var + eps) * gamma + beta),
            mean and variance over the pixels of a frame and the channels of a group
  linear    matrix product with bias, activation and residual (capi.linear):
            y = residual + act(x W^T + bias)
  grouped   the same over consecutive row groups of any sizes, each with a weight
            and bias of its own, the row offsets in device memory
            (capi.grouped_linear); rows in no group keep what the output held

Activations: none, gelu (erf), silu, gelu_tanh.  Inputs have the distributions
of the repository's benchmark: activations N(0, 1), weights N(0, 1 / fan-in);
a norm's channels have means and deviations of their own, as after a
convolution, and some means are many deviations large.
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPSILON = 1e-6


def listed():
    return [
        # The norm before the VAE's attention on the latent of a 64 x 64 thumbnail: a launch's latency.
        dict(name="norm_thumbnail", kind="norm", frames=1, pixels=64, channels=512, groups=32, pad=0,
             x="bf16", y="bf16", act="none"),
        # The same on one latent frame of a 720p video, 90 x 160 tokens.
        dict(name="norm_latent", kind="norm", frames=1, pixels=14400, channels=512, groups=32, pad=0,
             x="bf16", y="bf16", act="none"),
        # fp32 rows of a wider buffer, an odd picture, groups of 12 channels: a model of other widths.
        dict(name="norm_odd_fp32", kind="norm", frames=5, pixels=5757, channels=108, groups=9, pad=4,
             x="fp32", y="fp32", act="silu"),
        # A decoder residual block's norm and SiLU at full resolution, a slice of four 720p frames.
        dict(name="norm_decoder", kind="norm", frames=4, pixels=921600, channels=128, groups=32, pad=0,
             x="bf16", y="bf16", act="silu"),
        # One sampling step's timestep row to a block's six modulation vectors: reads its weight, hardly more.
        dict(name="linear_timestep", kind="linear", m=1, k=2560, n=15360, x="fp32", w="bf16", y="fp32",
             act="silu", bias=True, residual=False),
        # A prompt of odd length to the DiT's width, the other 16-bit type.
        dict(name="linear_text", kind="linear", m=77, k=5120, n=2560, x="fp16", w="fp16", y="fp16",
             act="none", bias=True, residual=False),
        # The VAE attention's out projection with the block's residual, one 720p latent frame.
        dict(name="linear_vae_out", kind="linear", m=14400, k=512, n=512, x="bf16", w="bf16", y="bf16",
             act="none", bias=True, residual=True),
        # The DiT's patch embedding of a 720p video: fp32 patches of 4 x 33 values.
        dict(name="linear_patches", kind="linear", m=21600, k=132, n=2560, x="fp32", w="bf16", y="bf16",
             act="none", bias=True, residual=False),
        # The 3B MLP's first product of the same video with its 64 text rows, tanh-GELU.
        dict(name="linear_mlp", kind="linear", m=21664, k=2560, n=10240, x="bf16", w="bf16", y="bf16",
             act="gelu_tanh", bias=True, residual=False),
        # A few tokens, one to a group, weights of many groups: a serving step.
        dict(name="grouped_tokens", kind="grouped", m=8, groups=32, sizes="spread", k=2048, n=1024,
             x="bf16", w="bf16", y="bf16", act="silu", bias=True, residual=False),
        # Ragged groups, some empty, and rows behind the last one: a batch of uneven requests.
        dict(name="grouped_ragged", kind="grouped", m=5000, groups=24, sizes="ragged", k=1000, n=1544,
             x="fp16", w="fp16", y="fp16", act="gelu", bias=True, residual=False),
        # The out projections of a DiT block whose video and text rows have weights of their own,
        # onto the fp32 residual stream.
        dict(name="grouped_streams", kind="grouped", m=21664, groups=2, sizes="streams", k=2560, n=2560,
             x="bf16", w="bf16", y="fp32", act="none", bias=True, residual=True),
    ]


def _between(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "grouped"])
    act = rng.choice(["none", "gelu", "silu", "gelu_tanh"])
    if kind == "norm":
        each, groups = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 24]), rng.choice([1, 2, 6, 8, 9, 16, 32])
        channels, frames = each * groups, rng.randint(1, 6)
        most = min(1 << 20, 100_000_000 // (channels * frames))
        return dict(kind="norm", frames=frames, pixels=_between(rng, 1, most), channels=channels,
                    groups=groups, pad=rng.choice([0, 0, 8, 3]), x=rng.choice(list(TYPES)),
                    y=rng.choice(list(TYPES)), act=act)
    k = _between(rng, 1, 6000) if rng.random() < 0.5 else 8 * _between(rng, 1, 700)
    n = _between(rng, 1, 6000) if rng.random() < 0.5 else 8 * _between(rng, 1, 700)
    x = rng.choice(list(TYPES))
    case = dict(kind=kind, k=k, n=n, x=x, w="fp16" if x == "fp16" else "bf16", y=rng.choice(list(TYPES)),
                act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.5)
    most = 6e11 / (2.0 * k * n)
    if kind == "linear":
        return dict(case, m=_between(rng, 1, int(max(1, min(16000, most)))))
    groups = _between(rng, 1, int(max(1, min(64, 5e8 // (2 * k * n)))))
    return dict(case, m=_between(rng, 1, int(max(1, min(16000, most)))), groups=groups,
                sizes=rng.choice(["spread", "ragged"]))


def _sizes(case):
    """Rows before the first group, then every group's: the case's alone, so that its work is known."""
    m, groups = case["m"], case["groups"]
    if case["sizes"] == "streams":   # 64 text rows behind the video's
        return 0, [m - 64, 64]
    if case["sizes"] == "spread":    # as even as can be, a row at most to a group where rows are few
        rows = [(i + 1) * m // groups - i * m // groups for i in range(groups)]
        return 0, rows
    r = random.Random(m * 64 + groups)
    share = [0.0 if r.random() < 0.2 else r.random() ** 3 for _ in range(groups)]
    first = m // 50
    scale = (m - first - m // 20) / (sum(share) or 1.0)   # a twentieth behind the last group
    return first, [int(s * scale) for s in share]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["kind"] == "norm":
        f, p, c = case["frames"], case["pixels"], case["channels"]
        mean, spread = normal(c), 0.5 + 2.0 * torch.rand(c, generator=gen, device="cuda")
        mean[:: max(2, c // 3)] *= 20.0
        wide = torch.empty(f, p, c + case["pad"], dtype=TYPES[case["x"]], device="cuda")
        for i in range(f):
            wide[i, :, :c] = normal(p, c) * spread + mean
        return dict(case=case, x=wide[:, :, :c], gamma=1.0 + 0.1 * normal(c), beta=0.1 * normal(c))
    m, k, n = case["m"], case["k"], case["n"]
    count = case.get("groups", 0)
    w = normal(max(1, count), n, k).mul_(k ** -0.5).to(TYPES[case["w"]])
    state = dict(case=case, x=normal(m, k).to(TYPES[case["x"]]), w=w if count else w[0], bias=None,
                 residual=None)
    if case["bias"]:
        state["bias"] = 0.1 * (normal(count, n) if count else normal(n))
    if case["residual"]:
        state["residual"] = normal(m, n).to(TYPES[case["y"]])
    if count:
        first, rows = _sizes(case)
        ends = [first]
        for r in rows:
            ends.append(ends[-1] + r)
        state["ends"] = ends   # the plain form's copy of the offsets
        state["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        state["out"] = normal(m, n).to(TYPES[case["y"]])
    return state


def _activate(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v * 0.5 ** 0.5)
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    return v


def _plain_norm(s):
    case, x = s["case"], s["x"]
    f, p, c, g = case["frames"], case["pixels"], case["channels"], case["groups"]
    x = x.float().reshape(f, p, g, c // g)
    x = x - x.mean(dim=(1, 3), keepdim=True)
    x = x / torch.sqrt((x * x).mean(dim=(1, 3), keepdim=True) + EPSILON)
    y = x.reshape(f, p, c) * s["gamma"] + s["beta"]
    return _activate(y, case["act"]).to(TYPES[case["y"]])


def _plain_linear(x, w, bias, residual, act):
    y = x.float() @ w.float().t()
    if bias is not None:
        y = y + bias
    y = _activate(y, act)
    return y if residual is None else y + residual.float()


def _plain_grouped(s):
    out, ends = s["out"], s["ends"]
    for g, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        if a < b:
            out[a:b] = _plain_linear(s["x"][a:b], s["w"][g], None if s["bias"] is None else s["bias"][g],
                                     None if s["residual"] is None else s["residual"][a:b],
                                     s["case"]["act"])
    return out


def run(state):
    case = state["case"]
    if own:
        from seedvr2_ncnn_amd import capi
        act = {"none": capi.ACT_NONE, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU,
               "gelu_tanh": capi.ACT_GELU_TANH}[case["act"]]
        out_type = TYPES[case["y"]]
        if case["kind"] == "norm":
            return capi.group_norm(state["x"], case["groups"], state["gamma"], state["beta"], EPSILON,
                                   act, out_dtype=out_type)
        if case["kind"] == "linear":
            return capi.linear(state["x"], state["w"], state["bias"], act, state["residual"],
                               out_dtype=out_type)
        return capi.grouped_linear(state["x"], state["offsets"], state["w"], state["bias"], act,
                                   state["residual"], out=state["out"])
    if case["kind"] == "norm":
        return _plain_norm(state)
    if case["kind"] == "linear":
        return _plain_linear(state["x"], state["w"], state["bias"], state["residual"],
                             case["act"]).to(TYPES[case["y"]])
    return _plain_grouped(state)


def work(case):
    if case["kind"] == "norm":
        values = case["frames"] * case["pixels"] * case["channels"]
        return {"bytes": values * (BYTES[case["x"]] + BYTES[case["y"]]) + 8 * case["channels"],
                "flops": 8 * values}
    m, k, n, weights = case["m"], case["k"], case["n"], 1
    if case["kind"] == "grouped":
        rows = _sizes(case)[1]
        m, weights = sum(rows), sum(r > 0 for r in rows)
    size = (m * k * BYTES[case["x"]] + weights * n * k * BYTES[case["w"]]
            + m * n * BYTES[case["y"]] * (2 if case["residual"] else 1)
            + (4 * weights * n if case["bias"] else 0))
    return {"bytes": max(1, size), "flops": 2 * m * k * n}


def _exact_activation(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":   # (1 + tanh u) / 2 = sigmoid(2 u)
        return v * torch.sigmoid(math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        count = case["pixels"] * (case["channels"] // case["groups"])
        frames = []
        for x in s["x"]:
            x = x.double()
            sums = x.sum(0).view(case["groups"], -1).sum(1, keepdim=True) / count
            x = x - sums.expand(-1, case["channels"] // case["groups"]).reshape(-1)
            var = x.square().sum(0).view(case["groups"], -1).sum(1, keepdim=True) / count
            scale = (var + EPSILON).rsqrt().expand(-1, case["channels"] // case["groups"]).reshape(-1)
            frames.append(_exact_activation(x * (scale * s["gamma"].double()) + s["beta"].double(),
                                            case["act"]))
        return torch.stack(frames)
    spans = [(0, case["m"], s["w"], s["bias"])]
    y = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
    if case["kind"] == "grouped":
        y = s["out"].double()
        ends = s["offsets"].tolist()
        spans = [(ends[g], ends[g + 1], s["w"][g], None if s["bias"] is None else s["bias"][g])
                 for g in range(case["groups"])]
    for a, b, w, bias in spans:
        v = torch.matmul(s["x"][a:b].double(), w.double().t().contiguous())
        v = _exact_activation(v if bias is None else v + bias.double(), case["act"])
        y[a:b] = v if s["residual"] is None else v + s["residual"][a:b].double()
    return y
