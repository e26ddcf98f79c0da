"""The operators of a channels-last pointwise block and the sizes at which they are measured.

  norm      group norm with an activation over channels-last positions (``group_norm_forward``)
  quant     each row of a matrix to 8-bit integers with a scale of its own (``quant_rows_forward``)
  product   matrix product of 8-bit integers with a scale for each row of either side, bias and activation
            (``inner_product_i8_forward``)

A block of a network runs them one after another: positions are normalised over groups of channels and activated, each
position's channels (a token) are quantised, and the pointwise product takes them with weights whose output channels were
quantised by the same row operator.

``own`` false computes the operators in elementary torch operations, ``own`` true calls the framework.
"""
import math

import torch

own = False

ACTS = ("none", "relu", "silu")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # one clip of an online step: the last trunk stage's 4 x 7 x 7 positions x 512 channels, where latency counts
        dict(name="norm one clip", op="norm", type="f32", n=1, s=196, c=512, groups=32, act="relu", ragged=False),
        # the first trunk stage of a 32-clip batch: 16 x 28 x 28 positions x 128 channels
        dict(name="norm trunk", op="norm", type="bf16", n=32, s=12544, c=128, groups=32, act="silu", ragged=False),
        # the stem's 56 x 56 x 64 output of 512 frames (32 clips x 16): more than the last-level cache holds
        dict(name="norm frames", op="norm", type="f32", n=512, s=3136, c=64, groups=16, act="relu", ragged=False),
        # padded clips of different lengths, a channel count that no vector width divides evenly into groups
        dict(name="norm ragged", op="norm", type="bf16", n=37, s=1571, c=210, groups=14, act="silu", ragged=True),
        # what "norm trunk" leaves, as the tokens of a pointwise product: many short rows
        dict(name="quant trunk", op="quant", type="bf16", m=401408, k=128),
        # long rows in full precision: weights by output channel, or the hidden rows of a wide layer
        dict(name="quant long", op="quant", type="f32", m=4096, k=8192),
        # the classifier of one clip: 512 features, 400 classes, where latency counts
        dict(name="product one clip", op="product", type="f32", m=1, n=400, k=512, bias=True, act="none"),
        # one token through a wide layer: the weights are all that is read
        dict(name="product one token", op="product", type="bf16", m=1, n=8192, k=8192, bias=False, act="none"),
        # a few tokens at a time, as a small serving batch has them
        dict(name="product few tokens", op="product", type="bf16", m=24, n=5120, k=4096, bias=True, act="silu"),
        # the pointwise product behind "quant trunk": many rows, short sums, as much written as computed
        dict(name="product pointwise", op="product", type="bf16", m=401408, n=128, k=128, bias=True, act="relu"),
        # odd sizes on every axis
        dict(name="product odd", op="product", type="f32", m=1003, n=777, k=1531, bias=True, act="relu"),
        # a long prompt through a wide layer: bound by the matrix cores
        dict(name="product large", op="product", type="bf16", m=8192, n=8192, k=8192, bias=True, act="none"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "quant", "product", "product", "product"))
    kind = rng.choice(("f32", "bf16"))
    if op == "norm":
        cg, groups = _log(rng, 1, 64), _log(rng, 1, 64)
        if rng.random() < 0.5:  # half of the draws are channel counts as networks have them
            cg, groups = 4 * _log(rng, 1, 16), rng.choice((8, 16, 32))
        c = cg * groups
        n = _log(rng, 1, 512)
        s = _log(rng, 1, max(1, min(16384, 90_000_000 // (n * c))))
        return dict(op=op, type=kind, n=n, s=s, c=c, groups=groups, act=rng.choice(ACTS), ragged=rng.random() < 0.3)
    if op == "quant":
        k = _log(rng, 1, 16384)
        return dict(op=op, type=kind, m=_log(rng, 1, min(400_000, 50_000_000 // k)), k=k)
    how = rng.choice(("tokens", "rows", "pointwise"))
    if how == "tokens":
        m, n, k = _log(rng, 1, 64), _log(rng, 64, 8192), _log(rng, 64, 8192)
    elif how == "rows":
        m, n, k = _log(rng, 65, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
    else:
        m, n, k = _log(rng, 8192, 400_000), _log(rng, 24, 512), _log(rng, 24, 512)
    if rng.random() < 0.6:  # most products have sizes that are multiples of a vector
        n, k = -(-n // 32) * 32, -(-k // 32) * 32
    return dict(op=op, type=kind, m=m, n=n, k=k, bias=rng.random() < 0.7, act=rng.choice(ACTS))


def _lengths(case):
    """Valid rows of each image of a ragged batch: spread from all to none, the same for every seed."""
    n, s = case["n"], case["s"]
    return [s - (s * ((7 * i) % n)) // max(1, n - 1) if n > 1 else (s + 1) // 2 for i in range(n)]


def _int8(shape, gen):
    """Quantised rows: a bell-shaped spread of which about one in a row reaches the largest code."""
    return (torch.randn(shape, generator=gen, device="cuda") * 36.0).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    uni = lambda *shape: torch.rand(shape, generator=gen, device="cuda")  # noqa: E731
    state, dt = dict(case), TYPES[case["type"]]
    if case["op"] == "norm":
        n, s, c = case["n"], case["s"], case["c"]
        # convolution outputs: channels of different spread and offset
        state["x"] = rand(n, s, c).mul_(0.5 + uni(c)).add_(rand(c)).to(dt)
        state["gamma"], state["beta"] = 1.0 + 0.2 * rand(c), 0.3 * rand(c)
        state["y"] = torch.full((n, s, c), 0.25, device="cuda", dtype=dt)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    elif case["op"] == "quant":
        m, k = case["m"], case["k"]
        x = rand(m, k).mul_(0.2 + uni(m, 1))
        x = (x * torch.sigmoid(x)).to(dt)  # activations of rows of different size
        if m > 2:
            x[1] = 0  # a padded token
        state["x"] = x
        state["q"] = torch.empty((m, k), dtype=torch.int8, device="cuda")
        state["scale"] = torch.empty(m, device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        state["x"], state["sx"] = _int8((m, k), gen), 0.002 + 0.03 * uni(m)
        state["w"], state["sw"] = _int8((n, k), gen), (0.2 + uni(n)) / (36.0 * math.sqrt(k))
        state["bias"] = 0.5 * rand(n) if case["bias"] else None
        state["y"] = torch.empty((m, n), dtype=dt, device="cuda")
    if own:
        _plan(state)
    return state


def _plan(state):
    """The plan and the workspace that a program keeps for these sizes."""
    from eco_amd import hip
    state["hip"], lib = hip, hip.load()
    state["lib"] = lib
    dt = {"f32": hip.DT_F32, "bf16": hip.DT_BF16}[state["type"]]
    state["dt"] = dt
    if state["op"] == "norm":
        state["plan"] = lib.group_norm_plan(state["n"], state["s"], state["c"], state["groups"], dt)
    elif state["op"] == "product":
        state["plan"] = lib.inner_product_i8_plan(state["m"], state["n"], state["k"], dt)
    size = state["plan"].ws_bytes if "plan" in state else 0
    state["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(state):
    lib, hip = state["lib"], state["hip"]
    stream = torch.cuda.current_stream().cuda_stream
    if state["op"] == "quant":
        lib.quant_rows_forward(_ptr(state["x"]), state["dt"], _ptr(state["q"]), _ptr(state["scale"]), state["m"], state["k"],
                               stream=stream)
        return {"q": state["q"], "scale": state["scale"]}
    act = {"none": hip.ACT_NONE, "relu": hip.ACT_RELU, "silu": hip.ACT_SILU}[state["act"]]
    if state["op"] == "norm":
        lib.group_norm_forward(state["plan"], _ptr(state["x"]), _ptr(state["gamma"]), _ptr(state["beta"]), _ptr(state["y"]),
                               eps=EPS, act=act, lengths=_ptr(state["lengths"]), workspace=_ptr(state["workspace"]),
                               stream=stream)
    else:
        lib.inner_product_i8_forward(state["plan"], _ptr(state["x"]), _ptr(state["sx"]), _ptr(state["w"]), _ptr(state["sw"]),
                                     _ptr(state["bias"]), _ptr(state["y"]), act=act, workspace=_ptr(state["workspace"]),
                                     stream=stream)
    return {"y": state["y"]}


def _activate(v, act):
    if act == "relu":
        return torch.clamp_min(v, 0.0)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _norm_plain(state):
    n, s, c, g = state["n"], state["s"], state["c"], state["groups"]
    x = state["x"].float().view(n, s, g, c // g)
    lengths = state["lengths"]
    if lengths is None:
        mean = x.mean(dim=(1, 3), keepdim=True)
        d = x - mean
        var = (d * d).mean(dim=(1, 3), keepdim=True)
    else:
        keep = (torch.arange(s, device=x.device)[None, :] < lengths[:, None]).view(n, s, 1, 1)
        count = (lengths.float() * (c // g)).clamp_min(1.0).view(n, 1, 1, 1)
        mean = torch.where(keep, x, 0.0).sum(dim=(1, 3), keepdim=True) / count
        d = x - mean
        var = torch.where(keep, d * d, 0.0).sum(dim=(1, 3), keepdim=True) / count
    v = (d / torch.sqrt(var + EPS)).view(n, s, c) * state["gamma"] + state["beta"]
    y = _activate(v, state["act"]).to(state["y"].dtype)
    if lengths is not None:  # rows behind an image's length stay as they were
        y = torch.where(keep.view(n, s, 1), y, state["y"])
    return {"y": y}


def _quant_plain(state):
    x = state["x"]
    top = x.float().abs().amax(dim=1, keepdim=True)
    # in 64 bits: a quotient next to a half must not go to the other integer
    q = torch.round(x.double() * 127.0 / torch.where(top > 0, top, 1.0).double()).to(torch.int8)
    return {"q": q, "scale": (top / 127.0).view(-1)}


def _product_plain(state):
    v = (state["x"].float() @ state["w"].float().t()) * state["sx"][:, None] * state["sw"]
    if state["bias"] is not None:
        v = v + state["bias"]
    return {"y": _activate(v, state["act"]).to(state["y"].dtype)}


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _norm_plain, "quant": _quant_plain, "product": _product_plain}[state["op"]](state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        rows = sum(_lengths(case)) if case["ragged"] else case["n"] * case["s"]
        # two for the mean, three for the variance, four for the result, and the activation
        return {"bytes": 2 * rows * case["c"] * size + 8 * case["c"], "flops": 10 * rows * case["c"]}
    if case["op"] == "quant":
        return {"bytes": case["m"] * case["k"] * (size + 1) + 4 * case["m"], "flops": 3 * case["m"] * case["k"]}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * k + n * k + 4 * (m + n * (2 if case["bias"] else 1)) + m * n * size, "flops": 2 * m * n * k}


def exact(case, seed):
    state = prepare(case, seed)
    act = {"none": lambda v: v, "relu": lambda v: v.clamp_min_(0.0), "silu": lambda v: v.mul_(torch.sigmoid(v))}
    if case["op"] == "norm":
        g, lengths = case["groups"], _lengths(case) if case["ragged"] else [case["s"]] * case["n"]
        out = state["y"].double()
        for i, rows in enumerate(lengths):
            if rows:
                z = state["x"][i, :rows].double().view(rows, g, -1).transpose(0, 1)
                var, mean = torch.var_mean(z, dim=(1, 2), unbiased=False, keepdim=True)
                z = ((z - mean) * (var + EPS).rsqrt()).transpose(0, 1).reshape(rows, -1)
                out[i, :rows] = act[case["act"]](z * state["gamma"].double() + state["beta"].double())
        return {"y": out}
    if case["op"] == "quant":
        scale = state["x"].double().abs().amax(dim=1) / 127.0
        return {"q": None, "scale": scale}
    y = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
    w = state["w"].double().t().contiguous()
    for a in range(0, case["m"], 65536):  # sums of products of 8-bit integers are exact in 64 bits
        b = min(a + 65536, case["m"])
        v = (state["x"][a:b].double() @ w) * state["sx"][a:b, None].double() * state["sw"].double()
        y[a:b] = act[case["act"]](v if state["bias"] is None else v + state["bias"].double())
    return {"y": y}
