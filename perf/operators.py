"""Measured cases of the 8-bit operators: rows quantised to 8-bit integers with a scale each, the
root-mean-square norm (with the residual's addition) that leaves such rows, and the matrix product of
two sets of such rows.

    q[r, k] = rint(127 x[r, k] / a[r]),  scale[r] = a[r] / 127,  a[r] = max_k |x[r, k]|
    norm:     x += residual;  h = x / sqrt(mean(x^2) + eps) * weight;  h in 8 bits as above
    product:  v[t, n] = (sum_k qx[t, k] qw[n, k]) sx[t] sw[n];  y = v, y += v or y = silu(gate) * up

A result in 8 bits is returned as the values it stands for (q times its scale, in the 16-bit type that
activations have in this package) beside its scales.
"""
import math

import torch

own = False

EPS = 1e-6
DEVICE = "cuda:0"
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # the attention's output of a decode step of eight sequences, before the O product
        {"name": "quantize_8x4096", "op": "quantize", "rows": 8, "width": 4096, "dtype": "bfloat16", "gap": 0},
        # the gated activations of a prompt, before the down product
        {"name": "quantize_2048x12288", "op": "quantize", "rows": 2048, "width": 12288, "dtype": "bfloat16", "gap": 0},
        # a gate and up weight when a model is loaded: a row is an output channel
        {"name": "quantize_weight", "op": "quantize", "rows": 24576, "width": 4096, "dtype": "bfloat16", "gap": 0},
        # one sequence decodes: the norm ahead of the q/k/v product
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "width": 4096, "dtype": "float32", "residual": "none"},
        # 64 sequences decode: the mixer's output is added on the way
        {"name": "norm_64x5120_residual", "op": "norm", "rows": 64, "width": 5120, "dtype": "float32",
         "residual": "float32"},
        # a long prompt
        {"name": "norm_8192x4096_residual", "op": "norm", "rows": 8192, "width": 4096, "dtype": "float32",
         "residual": "bfloat16"},
        # the fused q/k/v product of one decoding sequence
        {"name": "linear_1_qkv", "op": "linear", "tokens": 1, "inputs": 4096, "outputs": 6144, "mode": "store",
         "dtype": "float32"},
        # gate and up of a decode step of eight sequences
        {"name": "linear_8_gate_up", "op": "linear", "tokens": 8, "inputs": 4096, "outputs": 12288, "mode": "gated",
         "dtype": "bfloat16"},
        # down of a decode step of 64 sequences, added into the residual stream
        {"name": "linear_64_down", "op": "linear", "tokens": 64, "inputs": 12288, "outputs": 4096,
         "mode": "accumulate", "dtype": "float32"},
        # sizes that no tile divides
        {"name": "linear_333_odd", "op": "linear", "tokens": 333, "inputs": 2561, "outputs": 1111, "mode": "store",
         "dtype": "bfloat16"},
        # the q/k/v product of a prompt
        {"name": "linear_2048_qkv", "op": "linear", "tokens": 2048, "inputs": 4096, "outputs": 6144, "mode": "store",
         "dtype": "bfloat16"},
        # gate and up of several prompts in one step
        {"name": "linear_8192_gate_up", "op": "linear", "tokens": 8192, "inputs": 4096, "outputs": 12288,
         "mode": "gated", "dtype": "bfloat16"},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], even over its logarithm; half of the large ones a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n >= 256 and rng.random() < 0.5:
        n -= n % 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(("quantize", "norm", "linear", "linear"))
    if op == "quantize":
        width = _log(rng, 16, 32768)
        return {"op": op, "rows": _log(rng, 1, min(32768, (1 << 27) // width)), "width": width,
                "dtype": rng.choice(("bfloat16", "float32")), "gap": rng.choice((0, 0, 8, 13))}
    if op == "norm":
        width = _log(rng, 64, 16384)
        return {"op": op, "rows": _log(rng, 1, min(16384, (1 << 26) // width)), "width": width,
                "dtype": rng.choice(("float32", "float32", "bfloat16")),
                "residual": rng.choice(("none", "bfloat16", "float32"))}
    mode = rng.choice(("store", "accumulate", "gated"))
    tokens, inputs, outputs = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 64, 16384)
    while tokens * inputs * outputs > 1 << 38:  # under the largest listed case
        tokens = max(1, tokens // 2)
    dtype = {"store": rng.choice(("bfloat16", "float32")), "accumulate": "float32", "gated": "bfloat16"}[mode]
    return {"op": op, "tokens": tokens, "inputs": inputs, "outputs": outputs, "mode": mode, "dtype": dtype}


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _random_rows(gen, rows, width, std):
    """(8-bit integers, scales) of normally distributed rows; rows begin on multiples of 16 bytes."""
    x = _normal(gen, rows, width)
    a = x.abs().amax(1, keepdim=True)
    q = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.int8, device=DEVICE)[:, :width]
    q.copy_(torch.round(x * (127 / a)))
    return q, (a[:, 0] * (std / 127)).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    if case["op"] == "linear":
        m, k, n, gated = case["tokens"], case["inputs"], case["outputs"], case["mode"] == "gated"
        s["x"], s["x_scale"] = _random_rows(gen, m, k, 1.0)
        s["w"], s["w_scale"] = _random_rows(gen, 2 * n if gated else n, k, 1.0 / math.sqrt(k))
        s["y"] = _normal(gen, m, n).to(TYPES[case["dtype"]])
        if own:  # a user's program lays a weight out once
            from skyla_kernel_b200.kernels import ops
            s["weight"] = ops.Q8Weight(s["w"], s["w_scale"], gated=gated)
        return s
    rows, width = case["rows"], case["width"]
    # some channels of real activations are many times the others
    x = _normal(gen, rows, width) * torch.exp(0.7 * _normal(gen, width))
    if case["op"] == "quantize":
        s["x"] = torch.empty(rows, width + case["gap"], dtype=TYPES[case["dtype"]], device=DEVICE)[:, :width]
        s["x"].copy_(x)
        return s
    s["x"] = x.to(TYPES[case["dtype"]])
    s["weight"] = 1 + 0.1 * _normal(gen, width)
    if case["residual"] != "none":
        s["added"] = (0.3 * _normal(gen, rows, width)).to(TYPES[case["residual"]])
    return s


def _plain_rows(h):
    """Rows of 32-bit values in 8 bits: (the values they then stand for, scales)."""
    a = h.abs().amax(1, keepdim=True).double()
    q = torch.round(h.double() * 127 / a)  # in 64 bits: quotients that end in one half are common in 16-bit data
    scale = (a / 127).float()
    return (q.float() * scale).to(torch.bfloat16), scale[:, 0]


def _silu(v):
    return v / (1 + torch.exp(-v))


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    if s["op"] == "quantize":
        values, scale = _plain_rows(s["x"].float())
        return {"values": values, "scale": scale}
    if s["op"] == "norm":
        x = s["x"]
        if "added" in s:
            x.copy_(x.float() + s["added"].float())
        h = x.float()
        values, scale = _plain_rows(h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"])
        out = {"values": values, "scale": scale}
        if "added" in s:
            out["x"] = x
        return out
    v = (s["x"].float() @ s["w"].float().T) * s["x_scale"][:, None] * s["w_scale"]
    y = s["y"]
    if s["mode"] == "gated":
        n = s["outputs"]
        y.copy_(_silu(v[:, :n]) * v[:, n:])
    elif s["mode"] == "accumulate":
        y += v
    else:
        y.copy_(v)
    return y


def _run_own(s):
    from skyla_kernel_b200.kernels import ops
    if s["op"] == "linear":
        mode = {"store": ops.STORE, "accumulate": ops.ACCUMULATE, "gated": ops.GATED}[s["mode"]]
        return ops.linear_q8(ops.Q8Rows(s["x"], s["x_scale"]), s["weight"], s["y"], mode)
    if s["op"] == "quantize":
        rows = ops.quantize_rows(s["x"])
    else:
        rows = ops.rmsnorm_q8(s["x"], s["weight"], EPS, residual=s.get("added"))
    values = torch.empty(s["rows"], s["width"], dtype=torch.bfloat16, device=DEVICE)
    out = {"values": ops.dequantize_rows(rows, values), "scale": rows.scale}
    if "added" in s:
        out["x"] = s["x"]
    return out


def work(case):
    size = lambda name: TYPES[name].itemsize  # noqa: E731
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inputs"], case["outputs"]
        w = 2 * n if case["mode"] == "gated" else n
        moved = m * k + w * k + 4 * (m + w) + m * n * size(case["dtype"])
        if case["mode"] == "accumulate":
            moved += 4 * m * n
        return {"bytes": moved, "flops": 2 * m * w * k}
    rows, width = case["rows"], case["width"]
    # the values in, in 8 bits, and as what they stand for; the scales
    moved = rows * width * (size(case["dtype"]) + 1 + 2) + 4 * rows
    flops = 4 * rows * width
    if case["op"] == "norm":
        moved += 4 * width
        flops += 4 * rows * width
        if case["residual"] != "none":
            moved += rows * width * (size(case["dtype"]) + size(case["residual"]))
            flops += rows * width
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        k = case["inputs"]
        # whole numbers below 2^53: the sums are exact whatever their order
        acc = torch.matmul(s["x"].to(torch.float64), s["w"].to(torch.float64).t())
        v = torch.einsum("mn,m,n->mn", acc, s["x_scale"].to(torch.float64), s["w_scale"].to(torch.float64))
        assert k * 127 * 127 < 2 ** 53
        if case["mode"] == "gated":
            gate, up = v.chunk(2, dim=1)
            return torch.sigmoid(gate) * gate * up
        return s["y"].to(torch.float64) + v if case["mode"] == "accumulate" else v
    h = s["x"].to(torch.float64)
    out = {}
    if case["op"] == "norm":
        if "added" in s:
            h = h + s["added"].to(torch.float64)
            out["x"] = h
            h = h.to(TYPES[case["dtype"]]).to(torch.float64)  # the norm is that of the sum as it is kept
        h = h / (h.pow(2).sum(1, keepdim=True) / case["width"] + EPS).sqrt() * s["weight"].to(torch.float64)
    step = torch.linalg.vector_norm(h, ord=math.inf, dim=1) / 127
    return {**out, "scale": step, "values": (h / step[:, None]).round() * step[:, None]}
