"""What the 8-bit feed-forward operators are measured on: a root-mean-square norm (with the residual's
addition, and an output in 8 bits), the conversion to 8 bits with a scale for each block, the product
of 8-bit matrices with such scales, and the gated pair of projections with its activation.

Values in 8 bits are e4m3 (torch.float8_e4m3fn). A matrix is stored with its rows 16 bytes aligned;
an activation has one scale for each row and 128 columns, stored [blocks, rows]; a weight, [out, in],
one for each 128 x 128 block. With `own` false `run` computes in elementary torch operations; with
`own` true it makes the framework's calls on the same tensors.

Kinds of case and the ranges that `draw` takes them from:
* norm      1 .. 16384 rows of 64 .. 8192 columns, with or without residual and 8-bit output;
* quantize  1 .. 16384 rows of 64 .. 4096 columns, blocks of 1 x 128 or 128 x 128;
* gemm      C = A B^T (+ beta C0 + bias), m 1 .. 8192, n and k 64 .. 8192;
* gated     H = silu(A G^T) * (A U^T) in fp32 or 8 bits, m 1 .. 8192, n 64 .. 8192, k 64 .. 4096.
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0       # the largest e4m3 value
EPS = 1e-6
F8 = torch.float8_e4m3fn


def listed():
    return [
        # One token between two blocks of a decoder: latency.
        dict(name="norm_token", kind="norm", rows=1, cols=4096, residual=True, f8=True),
        # A ragged batch whose norm feeds an fp32 product.
        dict(name="norm_ragged", kind="norm", rows=4093, cols=1023, residual=False, f8=False),
        # A long prompt: the residual stream is read, updated and handed to an 8-bit product.
        dict(name="norm_prompt", kind="norm", rows=16384, cols=8192, residual=True, f8=True),
        # Activations of odd width on their way into an 8-bit product.
        dict(name="quantize_rows", kind="quantize", rows=2000, cols=1960, block_rows=1),
        # A large weight, converted when a model is loaded.
        dict(name="quantize_weight", kind="quantize", rows=16384, cols=4096, block_rows=128),
        # One token against a square weight, the residual added by the product.
        dict(name="gemm_token", kind="gemm", m=1, n=4096, k=4096, c0=True, bias=False),
        # A serving step of 32 sequences against a large weight.
        dict(name="gemm_few_rows", kind="gemm", m=32, n=16384, k=4096, c0=False, bias=True),
        # A layer of ragged sizes.
        dict(name="gemm_ragged", kind="gemm", m=4093, n=4099, k=1023, c0=False, bias=True),
        # A long prompt against a large weight.
        dict(name="gemm_prompt", kind="gemm", m=8192, n=8192, k=8192, c0=True, bias=False),
        # One token through the gated pair, handed on in 8 bits.
        dict(name="gated_token", kind="gated", m=1, n=10240, k=4096, f8=True),
        # A middle batch of odd sizes, handed on in fp32.
        dict(name="gated_ragged", kind="gated", m=1000, n=1960, k=1000, f8=False),
        # A long prompt through the gated pair, handed on in 8 bits.
        dict(name="gated_prompt", kind="gated", m=8192, n=10240, k=4096, f8=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quantize", "gemm", "gemm", "gemm", "gated", "gated"])
    if kind == "norm":
        return dict(kind="norm", rows=_log(rng, 1, 16384), cols=_log(rng, 64, 8192),
                    residual=rng.random() < 0.5, f8=rng.random() < 0.6)
    if kind == "quantize":
        return dict(kind="quantize", rows=_log(rng, 1, 16384), cols=_log(rng, 64, 4096),
                    block_rows=rng.choice([1, 128]))
    if kind == "gemm":
        return dict(kind="gemm", m=_log(rng, 1, 8192), n=_log(rng, 64, 8192),
                    k=_log(rng, 64, 8192), c0=rng.random() < 0.4, bias=rng.random() < 0.4)
    return dict(kind="gated", m=_log(rng, 1, 8192), n=_log(rng, 64, 8192), k=_log(rng, 64, 4096),
                f8=rng.random() < 0.6)


# ---- inputs -------------------------------------------------------------------------------------


def _blocks(size):
    return -(-size // BLOCK)


def _rows_of_bytes(rows, cols):
    """An e4m3 matrix whose rows are 16 bytes aligned."""
    return torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.uint8, device="cuda").view(F8)[:, :cols]


def _stored(x, block_rows):
    """x in 8 bits as a program keeps it: values with aligned rows, and the scales."""
    q, scales = _to_f8(x, block_rows)
    held = _rows_of_bytes(*x.shape)
    held.view(torch.uint8).copy_(q.view(torch.uint8))
    return held, scales


def _activations(gen, rows, cols):
    """Normal values with channels of differing size and a few of them far larger."""
    size = torch.exp(0.5 * torch.randn((cols,), generator=gen, device="cuda"))
    size[:: 61] *= 8
    return torch.randn((rows, cols), generator=gen, device="cuda") * size


def _weight(gen, n, k):
    return torch.randn((n, k), generator=gen, device="cuda") / math.sqrt(k)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = {"case": case}

    def empty(*shape):
        return torch.empty(shape, device="cuda")

    if kind in ("norm", "quantize"):
        rows, cols = case["rows"], case["cols"]
        state["x"] = _activations(gen, rows, cols)
        if kind == "norm":
            state["w"] = 1 + 0.2 * torch.randn((cols,), generator=gen, device="cuda")
            if case["residual"]:
                state["residual"] = 4 * _activations(gen, rows, cols)
                state["sum"] = empty(rows, cols)
        f8, block_rows = (case["f8"], 1) if kind == "norm" else (True, case["block_rows"])
    else:
        m, n, k = case["m"], case["n"], case["k"]
        rows, cols = m, n
        state["a"] = _stored(_activations(gen, m, k), 1)
        state["b"] = _stored(_weight(gen, n, k), 128)
        if kind == "gated":
            state["up"] = _stored(_weight(gen, n, k), 128)
            f8, block_rows = case["f8"], 1
        else:
            f8 = False
            if case["c0"]:
                state["c0"] = torch.randn((m, n), generator=gen, device="cuda")
            if case["bias"]:
                state["bias"] = torch.randn((n,), generator=gen, device="cuda")
    # The arrays that the program keeps for the results.
    if f8:
        state["q"] = _rows_of_bytes(rows, cols)
        state["q_scales"] = (empty(_blocks(cols), rows) if block_rows == 1
                             else empty(_blocks(rows), _blocks(cols)))
    else:
        state["out"] = empty(rows, cols)
    return state


# ---- the plain forms ----------------------------------------------------------------------------


def _to_f8(x, block_rows):
    """e4m3 values and fp32 scales of x: scale = max(largest magnitude / 448, 2^-126) of each block,
    value = x * (1 / scale) rounded to e4m3. Scales of rows come as [blocks, rows], of 128 x 128
    blocks as [row blocks, column blocks]."""
    rows, cols = x.shape
    nb, mb = _blocks(cols), -(-rows // block_rows)
    padded = torch.nn.functional.pad(x, (0, nb * BLOCK - cols, 0, mb * block_rows - rows))
    tiles = padded.view(mb, block_rows, nb, BLOCK)
    scale = (tiles.abs().amax(dim=(1, 3)) / TOP).clamp_min(2.0 ** -126)
    q = (tiles * (1 / scale)[:, None, :, None]).to(F8).view(torch.uint8)
    q = q.view(mb * block_rows, nb * BLOCK)[:rows, :cols].contiguous().view(F8)
    return q, (scale.t().contiguous() if block_rows == 1 else scale)


def _from_f8(stored, block_rows, dtype=torch.float32):
    """The matrix that 8-bit values and their scales stand for."""
    values, scales = stored
    rows, cols = values.shape
    if block_rows == 1:
        scale = scales.t()
    else:
        scale = scales.repeat_interleave(block_rows, 0)[:rows]
    return values.to(dtype) * scale.to(dtype).repeat_interleave(BLOCK, 1)[:, :cols]


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    out = {}
    if kind == "norm":
        t = state["x"]
        if case["residual"]:
            t = t + state["residual"]
            out["sum"] = t
        y = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * state["w"]
    elif kind == "quantize":
        y = state["x"]
    else:
        a = _from_f8(state["a"], 1)
        y = a @ _from_f8(state["b"], 128).t()
        if kind == "gated":
            y = y * torch.sigmoid(y) * (a @ _from_f8(state["up"], 128).t())
        else:
            if case["c0"]:
                y = y + state["c0"]
            if case["bias"]:
                y = y + state["bias"]
    if "q" in state:
        out["q"], out["q_scales"] = _to_f8(y, case.get("block_rows", 1))
    else:
        out["out"] = y
    return out


# ---- the framework's calls ----------------------------------------------------------------------

_STREAM = None


def _calls(state):
    """The framework's call on the state's tensors, its descriptor filled as a program fills it once
    for each layer."""
    import mensurflow_amd as mf

    global _STREAM
    if _STREAM is None:
        _STREAM = mf.Stream.wrap(torch.cuda.current_stream().cuda_stream)
    stream = _STREAM

    def array(t, dtype="float32"):
        return mf.DeviceArray.wrap(t.data_ptr(), tuple(t.shape), stream, dtype, t.stride())

    def matrix(values, scales, block_rows):
        s = array(scales)
        return mf.F8Matrix(array(values, "uint8"), s.T if block_rows == 1 else s, block_rows)

    def held(name):
        return array(state[name]) if name in state else None

    case = state["case"]
    kind = case["kind"]
    block_rows = case.get("block_rows", 1)
    q = matrix(state["q"], state["q_scales"], block_rows) if "q" in state else None
    if kind == "norm":
        desc = mf.rms_norm_desc(held("x"), held("w"), residual=held("residual"), eps=EPS,
                                summed=held("sum"), out=held("out"), out_f8=q)
        return lambda: mf.rms_norm_run(stream, desc)
    if kind == "quantize":
        x = held("x")
        return lambda: mf.quantize_f8(x, block_rows, out=q)
    up = matrix(*state["up"], 128) if kind == "gated" else None
    desc = mf.f8gemm_desc(matrix(*state["a"], 1), matrix(*state["b"], 128), up=up,
                          act=mf.ACT_SILU if up is not None else mf.ACT_NONE, c0=held("c0"),
                          beta=1.0 if "c0" in state else 0.0, bias=held("bias"), out=held("out"),
                          out_f8=q)
    return lambda: mf.f8gemm(stream, desc)


def run(state):
    if not own:
        return _plain(state)
    if "call" not in state:
        state["call"] = _calls(state)
    state["call"]()
    return {name: state[name] for name in ("sum", "q", "q_scales", "out") if name in state}


# ---- the work, and the results in 64 bits -------------------------------------------------------


def work(case):
    kind = case["kind"]

    def f8_bytes(rows, cols, block_rows=1):
        return rows * cols + 4 * -(-rows // block_rows) * _blocks(cols)

    if kind in ("norm", "quantize"):
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        if kind == "quantize":
            return {"bytes": 4 * n + f8_bytes(rows, cols, case["block_rows"]), "flops": 3 * n}
        made = f8_bytes(rows, cols) if case["f8"] else 4 * n
        return {"bytes": (12 if case["residual"] else 4) * n + 4 * cols + made,
                "flops": (7 if case["f8"] else 4) * n}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "gated":
        return {"bytes": f8_bytes(m, k) + 2 * f8_bytes(n, k, 128)
                + (f8_bytes(m, n) if case["f8"] else 4 * m * n), "flops": 4 * m * n * k}
    return {"bytes": f8_bytes(m, k) + f8_bytes(n, k, 128) + (8 if case["c0"] else 4) * m * n
            + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}


def _nearest_e4m3(v):
    """v (64 bits) on the grid of e4m3: 3 bits behind the leading one, least exponent -6, ties to
    even, at most 448."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_f8(y, block_rows):
    rows, cols = y.shape
    row = torch.arange(rows, device=y.device) // block_rows
    col = torch.arange(cols, device=y.device) // BLOCK
    by_col = torch.full((rows, _blocks(cols)), 0.0, dtype=torch.float64, device=y.device)
    by_col.scatter_reduce_(1, col.expand(rows, cols), y.abs(), "amax")
    top = torch.zeros((-(-rows // block_rows), _blocks(cols)), dtype=torch.float64, device=y.device)
    top.scatter_reduce_(0, row[:, None].expand(by_col.shape), by_col, "amax")
    scale = torch.maximum(top / TOP, torch.tensor(2.0 ** -126, dtype=torch.float64, device=y.device))
    q = _nearest_e4m3(y / scale[row][:, col])
    return q, (scale.t() if block_rows == 1 else scale)


def _exact_matrix(stored, block_rows):
    values, scales = stored
    rows, cols = values.shape
    row = torch.arange(rows, device=values.device)
    col = torch.arange(cols, device=values.device) // BLOCK
    s = scales.double()
    s = s[col][:, row].t() if block_rows == 1 else s[row // block_rows][:, col]
    return values.double() * s


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    out = {}
    if kind == "norm":
        t = state["x"].double()
        if case["residual"]:
            t = t + state["residual"].double()
            out["sum"] = t
        length = torch.sqrt((t * t).sum(1) / case["cols"] + EPS)
        y = t / length[:, None] * state["w"].double()
    elif kind == "quantize":
        y = state["x"].double()
    else:
        a = _exact_matrix(state["a"], 1)
        y = torch.mm(a, _exact_matrix(state["b"], 128).t())
        if kind == "gated":
            y = y / (1 + torch.exp(-y)) * torch.mm(a, _exact_matrix(state["up"], 128).t())
        else:
            if case["c0"]:
                y += state["c0"].double()
            if case["bias"]:
                y += state["bias"].double()
    if "q" in state:
        out["q"], out["q_scales"] = _exact_f8(y, case.get("block_rows", 1))
    else:
        out["out"] = y
    return out
