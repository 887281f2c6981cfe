"""What the 8-bit dense path and the log-probability operator are measured on.

A case is one call of one operator on inputs of a stated shape; ``run`` computes it either in plain
form (elementary torch operations in 32 bits, rounded once at the end) or, with ``own`` set, through
the package's public entry points.  The operators:

``quantize``   e4m3 codes of a bf16 matrix with one fp32 scale per block of ``block_rows`` x 128 values:
               ``a = max(max|x|, 2^-100)``, ``scale = a / 448``, ``code = e4m3(x * (448 / a))``
``norm``       ``h = bf16(delta + residual)``, ``y = h * rsqrt(mean(h^2) + eps) * (w + 1)``, ``y`` quantised
               by rows
``swiglu``     ``silu(z[:, :I]) * z[:, I:]``, quantised by rows
``gemm``       ``c[m, n] = sum over blocks t of 128: a_scale[m, t] * b_scale[n / 128, t] * (a . b over block t)``
``logprobs``   ``x[token] - lse(x)`` for a given token per row, the row's entropy, and its ``top`` most likely
               tokens (ties to the lowest id) with their log probabilities
"""
import math
import sys

import torch

own = False

FLOOR = 2.0 ** -100      # a block whose largest magnitude is below this is scaled as if it were this
TOP = 448.0              # largest e4m3 value
EPS = 1e-6
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # Attention output of a 4096-token prefill on its way into an 8-bit projection.
        {"name": "quantize rows 4096", "op": "quantize", "m": 4096, "k": 5120, "block_rows": 1},
        # A weight laid out once when a model is loaded (down projection).
        {"name": "quantize weight", "op": "quantize", "m": 5120, "k": 17408, "block_rows": 128},
        # One decoded token in front of gate_up: latency.
        {"name": "norm 1 token", "op": "norm", "m": 1, "k": 5120, "delta": True},
        # A long prefill in front of gate_up.
        {"name": "norm 8192 tokens", "op": "norm", "m": 8192, "k": 5120, "delta": True},
        # A handful of decoded tokens between gate_up and down: latency.
        {"name": "swiglu 7 tokens", "op": "swiglu", "m": 7, "k": 17408},
        # A prefill between gate_up and down.
        {"name": "swiglu 4096 tokens", "op": "swiglu", "m": 4096, "k": 17408},
        # One decoded token through gate_up: the weight is read once, nothing else counts.
        {"name": "gemm 1 token", "op": "gemm", "m": 1, "n": 34816, "k": 5120},
        # A ragged batch of decoded tokens through down.
        {"name": "gemm 77 tokens", "op": "gemm", "m": 77, "n": 5120, "k": 17408},
        # A prefill through gate_up: matrix-instruction rate.
        {"name": "gemm 4096 tokens", "op": "gemm", "m": 4096, "n": 34816, "k": 5120},
        # One decoded token over the vocabulary, with 20 alternatives: latency.
        {"name": "logprobs 1 row", "op": "logprobs", "m": 1, "v": 151936, "top": 20, "dtype": "float32", "masked": False},
        # Scores of a short answer over an odd vocabulary whose last ids are masked out.
        {"name": "logprobs 333 rows", "op": "logprobs", "m": 333, "v": 50257, "top": 5, "dtype": "float32", "masked": True},
        # Log probabilities of a whole 4096-token prompt, 20 alternatives at each position.
        {"name": "logprobs 4096 rows", "op": "logprobs", "m": 4096, "v": 151936, "top": 20, "dtype": "bfloat16", "masked": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "swiglu", "gemm", "gemm", "logprobs", "logprobs"])
    if op == "quantize":
        return {"op": op, "m": _log_int(rng, 1, 8192), "k": _log_int(rng, 16, 17408), "block_rows": rng.choice([1, 128])}
    if op == "norm":
        return {"op": op, "m": _log_int(rng, 1, 8192), "k": 8 * _log_int(rng, 8, 1024), "delta": rng.random() < 0.7}
    if op == "swiglu":
        return {"op": op, "m": _log_int(rng, 1, 4096), "k": 8 * _log_int(rng, 8, 2176)}
    if op == "gemm":
        return {"op": op, "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 16, 34816), "k": _log_int(rng, 64, 5120)}
    v = _log_int(rng, 64, 151936)
    return {"op": op, "m": _log_int(rng, 1, 4096), "v": v, "top": rng.choice([0, 1, 5, 20, 32]),
            "dtype": rng.choice(["bfloat16", "float16", "float32"]) if v < 75000 else "bfloat16",
            "masked": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _rows(shape, g, spread=0.5):
    """Activations: normal values whose columns differ in size, as a residual stream's channels do."""
    x = torch.randn(shape, generator=g, device="cuda")
    return x * torch.exp(spread * torch.randn(shape[-1], generator=g, device="cuda"))


def _bf16(t):
    return t.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"op": op}
    if op == "quantize":
        x = _rows((case["m"], case["k"]), g)
        s["x"] = _bf16(x * 0.02 if case["block_rows"] > 1 else x)
        s["block_rows"] = case["block_rows"]
    elif op == "norm":
        s["delta"] = _bf16(_rows((case["m"], case["k"]), g)) if case["delta"] else None
        s["residual"] = _bf16(3.0 * _rows((case["m"], case["k"]), g))
        s["weight"] = _bf16(0.1 * torch.randn(case["k"], generator=g, device="cuda"))
    elif op == "swiglu":
        s["z"] = _bf16(_rows((case["m"], 2 * case["k"]), g))
    elif op == "gemm":
        # codes and scales as the quantisers leave them: codes with rows of a multiple of 16 bytes,
        # the activation's scales with the rows contiguous
        a, sa = _quantize(_rows((case["m"], case["k"]), g), 1)
        b, sb = _quantize(0.02 * torch.randn((case["n"], case["k"]), generator=g, device="cuda"), 128)
        s["a"], s["b"] = _pitched(a), _pitched(b)
        s["a_scale"], s["b_scale"] = sa.t().contiguous().t(), sb.contiguous()
    else:
        m, v = case["m"], case["v"]
        x = 2.5 * torch.randn((m, v), generator=g, device="cuda")
        tokens = torch.randint(0, max(1, v * 15 // 16), (m,), generator=g, device="cuda")
        # most positions know their token, by a margin that differs from row to row
        x.scatter_add_(1, tokens[:, None], 14.0 * torch.rand((m, 1), generator=g, device="cuda"))
        if case["masked"]:
            x[:, max(1, v * 15 // 16):] = -math.inf
        s["logits"], s["tokens"], s["top"] = x.to(getattr(torch, case["dtype"])), tokens, case["top"]
    return s


def _pitched(q):
    m, k = q.shape
    out = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.uint8, device=q.device)
    out[:, :k] = q.view(torch.uint8)
    return out.view(E4M3)[:, :k]


# ------------------------------------------------------------------ plain form
def _blocked(x, rows):
    """(M, K) in blocks of rows x 128, zeros past the edges: (M / rows, rows, K / 128, 128)."""
    m, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 128, 0, -m % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def _quantize(x, rows):
    m, k = x.shape
    blocks = _blocked(x, rows)
    a = blocks.abs().amax((1, 3)).clamp_min(FLOOR)
    code = (blocks * torch.full_like(a, TOP).div(a)[:, None, :, None]).clamp(-TOP, TOP).to(E4M3)
    return code.view(-1, blocks.shape[2] * 128)[:m, :k], a / TOP


def _dequantize(q, scale, rows):
    m, k = q.shape
    wide = scale.repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]
    return q.float() * wide


def _order(x):
    """Whole numbers in the order of x's values (-0 and 0 alike)."""
    bits = (x + 0.0).view(torch.int32).long()
    return torch.where(bits >= 0, bits, -2147483648 - bits)


def _plain(s):
    op = s["op"]
    if op == "quantize":
        return _quantize(s["x"].float(), s["block_rows"])
    if op == "norm":
        h = s["residual"] if s["delta"] is None else (s["delta"].float() + s["residual"].float()).to(torch.bfloat16)
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * (s["weight"].float() + 1.0)
        return (*_quantize(y, 1), h)
    if op == "swiglu":
        gate, up = s["z"].float().chunk(2, -1)
        return _quantize(gate / (1.0 + torch.exp(-gate)) * up, 1)
    if op == "gemm":
        return (_dequantize(s["a"], s["a_scale"], 1) @ _dequantize(s["b"], s["b_scale"], 128).t()).to(torch.bfloat16)
    x = s["logits"].float()
    m, v = x.shape
    y = x - x.amax(-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(-1)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * y, 0.0).sum(-1) / total
    logprob = y.gather(1, s["tokens"][:, None])[:, 0] - lse
    del e
    key = (_order(x) << 32) - torch.arange(v, device=x.device)
    ids = (-torch.topk(key, min(s["top"], v), -1).values) & 0xFFFFFFFF
    return logprob, entropy, y.gather(1, ids) - lse[:, None], ids


# ------------------------------------------------------------------ the package's entry points
_package = None


def _ops():
    global _package
    if _package is None:
        sys.path.insert(0, "writes-that-matter_b200")
        from lcgemm import ops
        _package = ops
    return _package


def _own(s):
    ops, op = _package or _ops(), s["op"]
    if op == "quantize":
        return ops.quantize_fp8(s["x"], block_rows=s["block_rows"])
    if op == "norm":
        return ops.add_rmsnorm_fp8(s["delta"], s["residual"], s["weight"], EPS)
    if op == "swiglu":
        return ops.swiglu_fp8(s["z"])
    if op == "gemm":
        return ops.gemm_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"])
    return ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, m = case["op"], case["m"]
    if op == "logprobs":
        v, width = case["v"], {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
        return {"bytes": m * (v * width + 8 + 8 + 12 * case["top"]), "flops": 6 * m * v}
    k = case["k"]
    t = -(-k // 128)
    if op == "quantize":
        return {"bytes": 3 * m * k + 4 * -(-m // case["block_rows"]) * t, "flops": 3 * m * k}
    if op == "norm":
        return {"bytes": m * k * (7 if case["delta"] else 3) + 2 * k + 4 * m * t, "flops": 8 * m * k}
    if op == "swiglu":
        return {"bytes": 5 * m * k + 4 * m * t, "flops": 8 * m * k}
    n = case["n"]
    return {"bytes": m * k + n * k + 2 * m * n + 4 * t * (m + -(-n // 128)), "flops": 2 * m * n * k}


# ------------------------------------------------------------------ 64 bits
def _exact_codes(y, rows):
    """The scaled values before their rounding to e4m3, and the scales."""
    m, k = y.shape
    wide = torch.zeros((-(-m // rows) * rows, -(-k // 128) * 128), dtype=torch.float64, device=y.device)
    wide[:m, :k] = y
    cells = wide.unflatten(1, (-1, 128)).unflatten(0, (-1, rows))
    scale = torch.maximum(cells.abs().amax(dim=(1, 3)), torch.tensor(FLOOR, dtype=torch.float64, device=y.device)) / TOP
    return (cells / scale[:, None, :, None]).flatten(2, 3).flatten(0, 1)[:m, :k], scale


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "quantize":
        return _exact_codes(s["x"].double(), case["block_rows"])
    if op == "norm":
        r = s["residual"].double()
        total = r if s["delta"] is None else r + s["delta"].double()
        h = total.to(torch.bfloat16).double()            # the sum is kept in bf16, and that is what is normalised
        y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["k"] + EPS) * (1.0 + s["weight"].double())
        return (*_exact_codes(y, 1), total)
    if op == "swiglu":
        z = s["z"].double()
        half = case["k"]
        return _exact_codes(z[:, :half] * torch.sigmoid(z[:, :half]) * z[:, half:], 1)
    if op == "gemm":
        a, b = s["a"].to(torch.float64), s["b"].to(torch.float64)
        m, n, k = case["m"], case["n"], case["k"]
        col = torch.arange(k, device=a.device) // 128
        row = torch.arange(n, device=a.device) // 128
        a *= s["a_scale"].double()[:, col]
        b *= s["b_scale"].double()[row][:, col]
        return torch.matmul(a, b.transpose(0, 1))
    x = s["logits"].double()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    order = None
    if case["top"]:
        # ids of equal values in rising order: a stable sort of the values that can be among the first
        need = min(case["top"], case["v"])
        least = x.topk(need, -1).values[:, -1:]
        width = int((x >= least).sum(-1).max())
        near = torch.where(x >= least, torch.arange(case["v"], device=x.device), case["v"])
        near = near.topk(width, -1, largest=False, sorted=True).values
        held = torch.nn.functional.pad(x, (0, 1), value=-math.inf).gather(1, near)
        order = near.gather(1, torch.sort(held, dim=-1, descending=True, stable=True).indices[:, :need])
    else:
        order = torch.zeros((case["m"], 0), dtype=torch.long, device=x.device)
    return logp.gather(1, s["tokens"][:, None])[:, 0], entropy, logp.gather(1, order), order
