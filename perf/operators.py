"""The 8-bit integer path of a linear layer, as measurable cases: rows of activations to 8 bits with a scale a token (alone, and behind the RMS norm with
or without the residual's addition), and products of such rows with 8-bit weights that have a scale a channel (alone, and as the gate / up pair of a
feed-forward block).  The calls are those of the C ABI on caller-owned device buffers, as a host program makes them.

Formulas (rows t, columns c, output channels n):
  quant:  q = rint(127 x / a), a = max_c |x|, scale = a / 127
  norm:   h = round(x + residual), p = h w, q = rint(127 p / a), a = max_c |p|, scale = a / (127 sqrt(mean_c h^2 + eps))
  gemm:   out = round(xs[t] ws[n] sum_k xq[t, k] wq[n, k] + bias[n] + residual[t, n])
  pair:   out = round(g / (1 + exp(-g)) u), g and u products of the same rows with two tensors
A row of zeros has scale 0.
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5
LARGEST = 8192 * 14336 * 4096  # multiply-adds of the largest product


def listed():
    return [
        # decode: one token of an 8-billion-parameter decoder, ahead of its projections
        dict(name="norm 1", kind="norm", rows=1, cols=4096, dtype="bf16", residual=True),
        # one chunk of a long prompt
        dict(name="norm 8192", kind="norm", rows=8192, cols=4096, dtype="bf16", residual=True),
        # a decode batch, ahead of its down projections
        dict(name="quant 16", kind="quant", rows=16, cols=14336, dtype="bf16"),
        # three prompts of 1021 tokens ahead of the widest down projection, f16
        dict(name="quant 3063", kind="quant", rows=3063, cols=18944, dtype="f16"),
        # decode: query, key and value projections of one token, with their biases
        dict(name="gemm 1", kind="gemm", m=1, k=4096, n=6144, dtype="bf16", bias=True, residual=False),
        # a serving batch: its down projection, residual added
        dict(name="gemm 32 down", kind="gemm", m=32, k=14336, n=4096, dtype="bf16", bias=False, residual=True),
        # a serving batch: its logits in 32 bits
        dict(name="gemm 16 head", kind="gemm", m=16, k=3584, n=32000, dtype="f32", bias=False, residual=False),
        # a short question: down projection of 150 rows
        dict(name="gemm 150 down", kind="gemm", m=150, k=18944, n=3584, dtype="f16", bias=False, residual=True),
        # widths that no tile and no vector divides, rows that begin anywhere
        dict(name="gemm odd", kind="gemm", m=777, k=2741, n=1003, dtype="bf16", bias=True, residual=False),
        # one chunk of a long prompt: the largest product
        dict(name="gemm 8192 down", kind="gemm", m=8192, k=14336, n=4096, dtype="bf16", bias=False, residual=True),
        # the feed-forward pair of a small decode batch
        dict(name="pair 4", kind="pair", m=4, k=4096, n=14336, dtype="bf16"),
        # ... and of three prompts of 1021 tokens
        dict(name="pair 3063", kind="pair", m=3063, k=3584, n=18944, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """mostly what models have (multiples of 128 or of 16), some that nothing divides"""
    v, form = _log(rng, lo, hi), rng.random()
    return max(128, v // 128 * 128) if form < 0.55 else max(16, v // 16 * 16) if form < 0.8 else v


def draw(rng):
    kind = rng.choice(["norm", "quant", "gemm", "gemm", "gemm", "pair"])
    if kind in ("norm", "quant"):
        rows, cols = _log(rng, 1, 8192), _width(rng, 60, 16384 if kind == "norm" else 28672)
        rows = min(rows, max(1, 3063 * 18944 // cols))
        case = dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(["bf16", "bf16", "f16"]))
        if kind == "norm":
            case["residual"] = rng.random() < 0.7
        return case
    m, k, n = _log(rng, 1, 8192), _width(rng, 500, 18944), _width(rng, 200, 32000 if kind == "gemm" else 18944)
    m = min(m, max(1, LARGEST // (k * n * (2 if kind == "pair" else 1))))
    if kind == "pair":
        return dict(kind=kind, m=m, k=k, n=n, dtype=rng.choice(["bf16", "bf16", "f16"]))
    return dict(kind=kind, m=m, k=k, n=n, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), bias=rng.random() < 0.3, residual=rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)


def _randn(g, shape):
    return torch.randn(shape, generator=g, device="cuda")


def _activations(g, rows, cols, dtype):
    """normal values with a few channels far above the others, as a residual stream has them; of many rows some are padding, all zero"""
    x = _randn(g, (rows, cols))
    x *= 1.0 + 24.0 * (torch.rand((cols,), generator=g, device="cuda") < 0.004)
    if rows > 3:
        x *= (torch.rand((rows, 1), generator=g, device="cuda") > 0.01)
    return x.to(dtype)


def _codes(g, rows, cols):
    """rows of normal values in 8 bits with their scales: the largest of a row at 127"""
    x = _randn(g, (rows, cols))
    a = x.abs().amax(1, keepdim=True)
    return (x * (127.0 / a)).round_().to(torch.int8), (a[:, 0] / 127.0).contiguous()


def prepare(case, seed):
    g, dt = _gen(seed), DTYPE[case["dtype"]]
    s = dict(case=dict(case))
    if case["kind"] in ("norm", "quant"):
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(g, rows, cols, dt)
        s["q"] = torch.empty((rows, cols), dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty((rows,), device="cuda")
        if case["kind"] == "norm":
            s["weight"] = (1.0 + 0.1 * _randn(g, (cols,))).to(dt)
            if case["residual"]:
                s["residual"] = _activations(g, rows, cols, dt)
                s["h"] = torch.empty_like(s["x"])
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s["x"], s["xs"] = _codes(g, m, k)
    for name in ("w", "w2")[:2 if case["kind"] == "pair" else 1]:
        s[name], scales = _codes(g, n, k)
        s[name + "s"] = scales * k ** -0.5
    s["out"] = torch.empty((m, n), dtype=dt, device="cuda")
    if case.get("bias"):
        s["bias"] = _randn(g, (n,)).to(dt)
    if case.get("residual"):
        s["residual"] = _randn(g, (m, n)).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def _plain_codes(p, a):
    """p in 8 bits by its row's largest magnitude; the quotient in 64 bits, where a value next to a half decides as the definition does"""
    t = p.double() * 127.0 / a.double()[:, None]
    return torch.where(a[:, None] > 0, torch.round(t), 0.0).to(torch.int8)


def _plain_product(s, name):
    return s["x"].float() @ s[name].float().T * s["xs"][:, None] * s[name + "s"]


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "quant":
        p = s["x"].float()
        a = p.abs().amax(1)
        return dict(q=_plain_codes(p, a), scales=a / 127.0)
    if kind == "norm":
        h = s["x"]
        if case["residual"]:
            h = (s["x"].float() + s["residual"].float()).to(h.dtype)
        f = h.float()
        p = f * s["weight"].float()
        a = p.abs().amax(1)
        out = dict(q=_plain_codes(p, a), scales=a / 127.0 / torch.sqrt(f.square().mean(1) + EPS))
        if case["residual"]:
            out["h"] = h
        return out
    y = _plain_product(s, "w")
    if kind == "pair":
        y = y / (1.0 + torch.exp(-y)) * _plain_product(s, "w2")
    if case.get("bias"):
        y = y + s["bias"].float()
    if case.get("residual"):
        y = y + s["residual"].float()
    return y.to(DTYPE[case["dtype"]])


def run(s):
    if not own:
        return _plain(s)
    from vllm_rs_amd import _lib

    L, case, kind = _lib.load(), s["case"], s["case"]["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    dt = {"bf16": 0, "f16": 1, "f32": 2}[case["dtype"]]
    ptr = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    if kind in ("norm", "quant"):
        rows, cols = case["rows"], case["cols"]
        if kind == "quant":
            L.vra_quant_rows_i8(ptr("x"), ptr("q"), ptr("scales"), rows, cols, dt, stream)
        elif case["residual"]:
            L.vra_add_rms_norm_i8(ptr("x"), ptr("residual"), ptr("weight"), ptr("h"), ptr("q"), ptr("scales"), rows, cols, EPS, dt, stream)
            return dict(q=s["q"], scales=s["scales"], h=s["h"])
        else:
            L.vra_rms_norm_i8(ptr("x"), ptr("weight"), ptr("q"), ptr("scales"), rows, cols, EPS, dt, stream)
        return dict(q=s["q"], scales=s["scales"])
    if "workspace" not in s:  # one for all products of a stream, zeroed once
        s["workspace"] = torch.zeros((L.vra_w8a8_workspace_bytes(),), dtype=torch.uint8, device="cuda")
    m, k, n = case["m"], case["k"], case["n"]
    if kind == "pair":
        L.vra_w8a8_gate_up_silu(ptr("x"), ptr("xs"), ptr("w"), ptr("ws"), ptr("w2"), ptr("w2s"), ptr("out"), ptr("workspace"), m, k, n, dt, stream)
    else:
        L.vra_w8a8_gemm(ptr("x"), ptr("xs"), ptr("w"), ptr("ws"), ptr("bias"), ptr("residual"), ptr("out"), ptr("workspace"), m, k, n, dt, stream)
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("norm", "quant"):
        rows, cols = case["rows"], case["cols"]
        elements = rows * cols
        if case["kind"] == "quant":
            return dict(bytes=elements * (size + 1) + 4 * rows, flops=4 * elements)
        return dict(bytes=elements * (size * (3 if case["residual"] else 1) + 1) + size * cols + 4 * rows, flops=8 * elements)
    m, k, n = case["m"], case["k"], case["n"]
    tensors = 2 if case["kind"] == "pair" else 1
    moved = m * k + 4 * m + tensors * (n * k + 4 * n) + size * m * n
    moved += size * n * bool(case.get("bias")) + size * m * n * bool(case.get("residual"))
    return dict(bytes=moved, flops=2 * tensors * m * n * k)


# ---------------------------------------------------------------------------------------------------------------- the definition in 64 bits
def _row_codes64(v):
    top = v.abs().max(dim=1, keepdim=True).values
    safe = torch.where(top == 0, torch.ones_like(top), top)
    return (127.0 * v / safe).round().to(torch.int8), top.squeeze(1) / 127.0


def _dot64(s, name):
    x, rows = s["x"].to(torch.float64), []
    for part in s[name].split(4096):  # output channels by blocks: the 64-bit copies stay small
        rows.append(x.matmul(part.to(torch.float64).t().contiguous()))
    return torch.cat(rows, 1) * torch.outer(s["xs"].to(torch.float64), s[name + "s"].to(torch.float64))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        q, scales = _row_codes64(s["x"].to(torch.float64))
        return dict(q=q, scales=scales)
    if case["kind"] == "norm":
        x = s["x"].to(torch.float64)
        if case["residual"]:  # the sum is stored, and normed as it is stored
            h = x + s["residual"].to(torch.float64)
            x = h.to(DTYPE[case["dtype"]]).to(torch.float64)
        q, top = _row_codes64(x * s["weight"].to(torch.float64))
        out = dict(q=q, scales=top * torch.rsqrt((x * x).sum(1) / case["cols"] + EPS))
        if case["residual"]:
            out["h"] = h
        return out
    y = _dot64(s, "w")
    if case["kind"] == "pair":
        return y * torch.sigmoid(y) * _dot64(s, "w2")
    for name in ("bias", "residual"):
        if name in s:
            y = y + s[name].to(torch.float64)
    return y
