"""The dense operators around a sparse-pooling layer, as cases that can be timed and compared.

Three operators: ``linear_act`` (matrix product with bias, activation and residual), ``group_norm_act``
(channels-last group norm with an activation) and 8-bit activation checkpoints (``encode_activation`` /
``decode_activation``, and ``checkpoint="int8"`` of the other two, whose backward passes read them).  With ``own``
true ``run`` makes the framework's public calls; with ``own`` false it computes the same with elementary torch
operations in 32 bits, rounded once at the end.  ``exact`` restates the definitions in 64 bits.
"""
import math

import torch

own = False

BLOCK = 32                       # channels that share one exponent of an 8-bit checkpoint
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def _linear(name, mode, dtype, M, K, N, act, ckpt="none"):
    return dict(name=name, op="linear", mode=mode, dtype=dtype, M=M, K=K, N=N, act=act, ckpt=ckpt)


def _norm(name, mode, dtype, samples, positions, channels, groups, act, ckpt="none"):
    return dict(name=name, op="norm", mode=mode, dtype=dtype, samples=samples, positions=positions,
                channels=channels, groups=groups, act=act, ckpt=ckpt)


def _codec(name, dtype, rows, channels):
    return dict(name=name, op="codec", mode="infer", dtype=dtype, rows=rows, channels=channels)


def listed():
    return [
        # one token through a projection at the layer's width: serving, where latency counts
        _linear("linear_token_bf16", "infer", "bf16", 1, 4096, 4096, "gelu"),
        # the same with the framework's default parameters (fp32), to the 2048 outputs of the Cover-TopK16 layer
        _linear("linear_token_f32", "infer", "f32", 1, 4096, 2048, "silu"),
        # a ragged serving batch
        _linear("linear_few_bf16", "infer", "bf16", 37, 4096, 4096, "identity"),
        # a training step at the headline batch and width
        _linear("linear_train_bf16", "train", "bf16", 1024, 4096, 4096, "gelu"),
        # a training step with fp32 parameters
        _linear("linear_train_f32", "train", "f32", 1024, 4096, 2048, "gelu"),
        # rows that no vector load or tile divides
        _linear("linear_ragged_bf16", "train", "bf16", 777, 1001, 515, "relu"),
        # the Mode-B batch, with the input and the activation's derivative kept in 8 bits
        _linear("linear_ckpt_bf16", "train", "bf16", 8192, 4096, 4096, "gelu", "int8"),
        # one token's norm before a projection
        _norm("norm_token_bf16", "infer", "bf16", 1, 1, 4096, 32, "identity"),
        # token rows (each token its own statistics) of the headline batch, fp32
        _norm("norm_rows_f32", "train", "f32", 1024, 1, 4096, 64, "gelu"),
        # channels-last maps of 64 x 64 positions
        _norm("norm_maps_bf16", "train", "bf16", 16, 4096, 512, 32, "silu"),
        # odd maps with an 8-bit checkpoint of the input
        _norm("norm_ckpt_bf16", "train", "bf16", 12, 777, 1000, 8, "gelu", "int8"),
        # an activation of the Mode-B batch written to 8 bits and read back
        _codec("codec_f32", "f32", 8192, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd(rng, v, step):
    """Half of the sizes are multiples of `step`, the others as they fall."""
    return max(step, v // step * step) if rng.random() < 0.5 else v


def draw(rng):
    dtype = rng.choice(["bf16", "f32"])
    kind = rng.choice(["linear", "linear", "norm", "norm", "codec"])
    # relu's and the 8-bit derivative's jumps turn a last-bit difference of z into a whole step of the gradient,
    # so fp32 training draws keep to what is continuous there
    if kind == "linear":
        mode = rng.choice(["infer", "train"])
        M = _log(rng, 1, 8192)
        K, N = _odd(rng, _log(rng, 16, 8192), 64), _odd(rng, _log(rng, 16, 8192), 64)
        while M * K * N > 2 ** 34:
            M = max(1, M // 2)
        ckpt = rng.choice(["none", "int8"]) if mode == "train" else "none"
        acts = ["identity", "relu", "gelu", "silu"]
        if dtype == "f32" and mode == "train":
            acts = ["identity"] if ckpt == "int8" else ["identity", "gelu", "silu"]
        return dict(op="linear", mode=mode, dtype=dtype, M=M, K=K, N=N, act=rng.choice(acts), ckpt=ckpt)
    if kind == "norm":
        mode = rng.choice(["infer", "train"])
        groups = rng.choice([1, 2, 4, 8, 16, 32, 64])
        channels = groups * _log(rng, 4, 4096 // groups)
        samples, positions = _log(rng, 1, 1024), _log(rng, 1, 4096)
        while samples * positions * channels > 2 ** 24:
            positions, samples = max(1, positions // 2), max(1, samples * 3 // 4)
        ckpt = rng.choice(["none", "int8"]) if mode == "train" else "none"
        acts = ["identity", "gelu", "silu"] + (["relu"] if dtype == "bf16" or mode == "infer" else [])
        return dict(op="norm", mode=mode, dtype=dtype, samples=samples, positions=positions, channels=channels,
                    groups=groups, act=rng.choice(acts), ckpt=ckpt)
    rows, channels = _log(rng, 1, 8192), _odd(rng, _log(rng, 1, 8192), 32)
    while rows * channels > 2 ** 25:
        rows = max(1, rows // 2)
    return dict(op="codec", mode="infer", dtype=dtype, rows=rows, channels=channels)


# ---------------------------------------------------------------- inputs

def _inputs(case, seed):
    """The tensors of a case on the GPU.  Inputs have channels of unlike size, as activations do."""
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).add_(mean)

    def channels(n):
        return torch.exp(0.5 * torch.randn(n, generator=gen, device=dev))

    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s = dict(x=normal(M, K).mul_(channels(K)), w=normal(N, K, scale=K ** -0.5), b=normal(N, scale=0.1),
                 r=normal(M, N))
        if case["mode"] == "train":
            s["dy"] = normal(M, N, scale=0.1)
    elif case["op"] == "norm":
        S, P, C = case["samples"], case["positions"], case["channels"]
        s = dict(x=normal(S, P, C).mul_(channels(C)).add_(normal(C, scale=0.5)), w=normal(C, scale=0.1, mean=1.0),
                 b=normal(C, scale=0.1))
        if case["mode"] == "train":
            s["dy"] = normal(S, P, C, scale=0.1)
    else:
        s = dict(x=normal(case["rows"], case["channels"]).mul_(channels(case["channels"])))
    return {k: v.to(dt) for k, v in s.items()}


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["mode"] == "train":
        for k in ("x", "w", "b", "r"):
            if k in s:
                s[k].requires_grad_(True)
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------- plain forms (32 bits)

def _act(z, act):
    if act == "identity":
        return z
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    return z / (1 + torch.exp(-z))


def _dact(z, act):
    if act == "identity":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _read_back(x):
    """What an 8-bit checkpoint of x [..., C] reads back as: per 32 channels the smallest power of two s with
    max |x| <= 127 s, whole multiples of s."""
    C = x.shape[-1]
    pad = -C % BLOCK
    v = torch.nn.functional.pad(x, (0, pad)).reshape(*x.shape[:-1], -1, BLOCK)
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    s = torch.ldexp(torch.ones_like(m), torch.where(m <= 127 / 128, e - 7, e - 6).clamp(min=-126))
    return (torch.round(v / s) * s).reshape(*x.shape[:-1], C + pad)[..., :C]


def _read_back_slope(d):
    """What the 8-bit code of an activation's derivative reads back as: multiples of 1/192 from -32/192 on."""
    return (torch.round(d * 192).clamp(-32, 223)) / 192


def _plain_linear(case, x, w, b, r, dy):
    z = x @ w.t() + b
    out = dict(y=_act(z, case["act"]) + r)
    if dy is not None:
        d = _dact(z, case["act"])
        if case["ckpt"] == "int8":
            x, d = _read_back(x), _read_back_slope(d)
        dz = dy * d
        out.update(dx=dz @ w, dw=dz.t() @ x, db=dz.sum(0), dr=dy)
    return out


def _plain_norm(case, x, w, b, dy):
    S, P, C = x.shape
    G = case["groups"]

    def spread(t):                       # [S, G] -> [S, 1, C]
        return t.repeat_interleave(C // G, 1)[:, None]

    def mean(t):                         # over the positions and channels of a group
        return t.reshape(S, P, G, C // G).mean((1, 3))

    mu = mean(x)
    var = mean((x - spread(mu)) ** 2)
    rstd = 1 / torch.sqrt(var + 1e-5)
    out = dict(y=_act((x - spread(mu)) * spread(rstd) * w + b, case["act"]))
    if dy is not None:
        if case["ckpt"] == "int8":
            x = _read_back(x)
        h = (x - spread(mu)) * spread(rstd)
        du = dy * _dact(h * w + b, case["act"])
        dh = du * w
        dx = (dh - spread(mean(dh)) - h * spread(mean(dh * h))) * spread(rstd)
        out.update(dx=dx, dw=(du * h).sum((0, 1)), db=du.sum((0, 1)))
    return out


def _plain(case, s, dtype):
    """All outputs of a case in `dtype`, from the inputs `s`."""
    t = {k: v.detach().to(dtype) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "linear":
        return _plain_linear(case, t["x"], t["w"], t["b"], t["r"], t.get("dy"))
    if case["op"] == "norm":
        return _plain_norm(case, t["x"], t["w"], t["b"], t.get("dy"))
    return dict(back=_read_back(t["x"]))


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if not own:
        dt = DTYPES[case["dtype"]]
        with torch.no_grad():
            return {k: v.to(dt) for k, v in _plain(case, state, torch.float32).items()}
    import granulelayer_b200 as gl

    if case["op"] == "codec":
        return dict(back=gl.decode_activation(gl.encode_activation(state["x"])))
    if case["op"] == "linear":
        args = (state["x"], state["w"], state["b"], state["r"])
        call, kw = gl.linear_act, dict(activation=case["act"])
    else:
        args = (state["x"], case["groups"], state["w"], state["b"])
        call, kw = gl.group_norm_act, dict(activation=case["act"], eps=1e-5)
    if case["mode"] == "infer":
        with torch.no_grad():
            return dict(y=call(*args, **kw))
    y = call(*args, checkpoint=case["ckpt"], **kw)
    names = ("x", "w", "b", "r") if case["op"] == "linear" else ("x", "w", "b")
    grads = torch.autograd.grad(y, [state[n] for n in names], state["dy"])
    return dict(y=y.detach(), **{"d" + n: g for n, g in zip(names, grads)})


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    e = DTYPES[case["dtype"]].itemsize
    train, ckpt = case["mode"] == "train", case.get("ckpt") == "int8"
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        # forward: x, w, b, residual in, y out; backward: dy in, dx, dw, db out (dr is dy itself)
        nbytes = e * (M * K + N * K + N + 2 * M * N)
        if train:
            nbytes += e * (M * N + M * K + N * K + N)
        return {"bytes": nbytes, "flops": 2 * M * N * K * (3 if train else 1)}
    if case["op"] == "norm":
        n, C = case["samples"] * case["positions"] * case["channels"], case["channels"]
        nbytes = e * (2 * n + 2 * C) + (e * (2 * n + 2 * C) if train else 0)   # x, y; dy, dx; parameters, gradients
        return {"bytes": nbytes, "flops": n * ((25 if train else 8) + (6 if ckpt else 0))}
    n = case["rows"] * case["channels"]
    kept = n + case["rows"] * -(-case["channels"] // BLOCK)                     # codes and exponents: written, read
    return {"bytes": 2 * n * e + 2 * kept, "flops": 6 * n}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_act(z, act):
    """(act(z), act'(z)) in 64 bits."""
    if act == "identity":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
    if act == "gelu":
        cdf = torch.special.erfc(-z / math.sqrt(2)) / 2
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    sig = torch.sigmoid(z)
    return z * sig, sig + z * sig * torch.sigmoid(-z)


def _exact_blocks(x):
    """Checkpoint blocks by their definition: a scale 2^e per 32 channels, found by counting up from the largest
    power that is too small."""
    out = torch.empty_like(x)
    for c0 in range(0, x.shape[-1], BLOCK):
        v = x[..., c0:c0 + BLOCK]
        top = v.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149) / 127)) - 1
        for _ in range(3):
            e = torch.where(top > 127 * torch.exp2(e), e + 1, e)
        s = torch.exp2(e.clamp(min=-126))
        out[..., c0:c0 + BLOCK] = torch.round(v / s) * s
    return out


def exact(case, seed):
    s = {k: v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "codec":
        return dict(back=_exact_blocks(s["x"]))
    if case["op"] == "linear":
        z = torch.einsum("mk,nk->mn", s["x"], s["w"]) + s["b"]
        a, slope = _exact_act(z, case["act"])
        out = dict(y=a + s["r"])
        if case["mode"] == "train":
            x = s["x"]
            if case["ckpt"] == "int8":
                x = _exact_blocks(x)
                slope = torch.round(slope * 192) / 192
            g = s["dy"] * slope
            out.update(dx=torch.einsum("mn,nk->mk", g, s["w"]), dw=torch.einsum("mn,mk->nk", g, x),
                       db=torch.einsum("mn->n", g), dr=s["dy"])
        return out
    S, P, C = s["x"].shape
    G = case["groups"]

    def split(t):
        return t.reshape(S, P, G, C // G)

    x, gam, bet = split(s["x"]), s["w"].reshape(G, -1), s["b"].reshape(G, -1)
    var, mu = torch.var_mean(x, dim=(1, 3), correction=0, keepdim=True)
    sd = torch.sqrt(var + 1e-5)
    a, _ = _exact_act((x - mu) / sd * gam + bet, case["act"])
    out = dict(y=a.reshape(S, P, C))
    if case["mode"] == "train":
        if case["ckpt"] == "int8":
            x = split(_exact_blocks(s["x"]))
        h = (x - mu) / sd
        _, slope = _exact_act(h * gam + bet, case["act"])
        du = split(s["dy"]) * slope
        q = du * gam
        dx = (q - q.mean((1, 3), keepdim=True) - h * (q * h).mean((1, 3), keepdim=True)) / sd
        out.update(dx=dx.reshape(S, P, C), dw=(du * h).sum((0, 1)).reshape(C), db=du.sum((0, 1)).reshape(C))
    return out
