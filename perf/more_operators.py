"""Root-mean-square norm with the residual's addition, its form with 8-bit results, rows in 8 bits and back, and the matrix
product of 8-bit integers, as cases that can be timed and whose outputs can be compared.

    h = round(x + residual),   y = h r w,   r = 1 / sqrt(mean(h^2) + eps)     (over the last dimension; w or 1 + w)
    scale = max|y| / 127,   q = round(y / scale)                              (of each row)
    C[m, n] = sum_k A[m, k] B[n, k] a_scale[m] b_scale[n] + bias[n]           (A, B int8)

Sizes follow the repository's layer (hidden size 2048, 32 value heads of 128, the in-projection's 12352 columns and their
1544 on one of eight GPUs); row counts run from one decoded token to a block of 4 x 32768 tokens.  ``run`` computes each
operator in elementary operations in 32 bits, or, where ``own`` is true, through the framework's entry points.  Rows in
8 bits are returned as the values they stand for.  Inputs are made on the GPU from the seed alone.
"""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_OPS = 2 * 131072 * 12352 * 2048  # of the largest listed product
MOST_ELEMENTS = 131072 * 2048         # of the largest listed norm


def listed():
    return [
        # the norm in front of a layer for one user's token: the smallest call, all latency
        {"name": "norm_one", "kind": "norm", "rows": 1, "n": 2048, "dtype": "bf16", "wdtype": "bf16", "residual": True, "plus_one": True},
        # the same for the block's 4 sequences of 32768 tokens
        {"name": "norm_block", "kind": "norm", "rows": 131072, "n": 2048, "dtype": "bf16", "wdtype": "fp32", "residual": True, "plus_one": False},
        # its gradients in a training step of 2 x 4096 tokens, the residual's gradient added
        {"name": "norm_grad", "kind": "norm_grad", "rows": 8192, "n": 2048, "dtype": "bf16", "wdtype": "fp32", "residual": True, "plus_one": False},
        # the same in 32 bits at an odd width, without a residual
        {"name": "norm_grad_odd", "kind": "norm_grad", "rows": 1001, "n": 1409, "dtype": "fp32", "wdtype": "fp32", "residual": False, "plus_one": True},
        # a long prompt's norm with 8-bit rows, and the values they stand for
        {"name": "norm8_prefill", "kind": "norm8", "rows": 32768, "n": 2048, "dtype": "bf16", "wdtype": "bf16", "residual": True, "plus_one": True},
        # the decode step of 64 sequences up to the convolution: norm to 8 bits, in-projection in 8 bits
        {"name": "project_decode", "kind": "project", "m": 64, "n": 12352, "k": 2048, "dtype": "bf16"},
        # the head outputs of 8192 tokens in front of the output projection
        {"name": "quant_tokens", "kind": "quant", "rows": 8192, "n": 4096, "dtype": "bf16"},
        # the in-projection's weights as they are loaded, from 32 bits
        {"name": "quant_weights", "kind": "quant", "rows": 12352, "n": 2048, "dtype": "fp32"},
        # one user's token through the in-projection: the weights' bytes
        {"name": "gemm8_one", "kind": "gemm8", "m": 1, "n": 12352, "k": 2048, "out": "bf16", "bias": False},
        # a short prompt of odd length on one of eight GPUs, odd depth, with a bias
        {"name": "gemm8_ragged", "kind": "gemm8", "m": 1003, "n": 1544, "k": 1999, "out": "fp16", "bias": True},
        # the output projection of a prompt's 8192 tokens, into a 32-bit residual stream
        {"name": "gemm8_out", "kind": "gemm8", "m": 8192, "n": 2048, "k": 4096, "out": "fp32", "bias": False},
        # the block's in-projection at its largest
        {"name": "gemm8_block", "kind": "gemm8", "m": 131072, "n": 12352, "k": 2048, "out": "bf16", "bias": False},
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "norm8", "quant", "gemm8", "gemm8", "gemm8", "project"])
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("gemm8", "project"):
        n = rng.choice([12352, 1544, 2048, 4096]) if rng.random() < 0.5 else _log_int(rng, 8, 16384)
        k = rng.choice([2048, 4096, 512]) if rng.random() < 0.5 else _log_int(rng, 32, 8192)
        m = _log_int(rng, 1, max(1, min(131072, MOST_OPS // (2 * n * k))))
        if kind == "project":
            return {"kind": kind, "m": min(m, 32768), "n": n, "k": k, "dtype": dt}
        return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "bias": rng.random() < 0.4}
    n = rng.choice([64, 1000, 2048, 4096, 8192]) if rng.random() < 0.6 else _log_int(rng, 17, 16384)
    most = MOST_ELEMENTS // n // (1 if kind == "norm" else 4)
    rows = _log_int(rng, 1, min(131072, most // 2 if dt == "fp32" else most))
    if kind == "quant":
        return {"kind": kind, "rows": rows, "n": n, "dtype": dt}
    return {"kind": kind, "rows": rows, "n": n, "dtype": dt, "wdtype": rng.choice(["fp32", dt]), "residual": rng.random() < 0.7,
            "plus_one": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _hidden(gen, rows, n, dt):
    """Rows as a residual stream has them: a few channels are far larger than the others."""
    channel = torch.exp(0.5 * torch.randn(n, generator=gen, device=DEV))
    channel[torch.randint(0, n, (max(1, n // 256),), generator=gen, device=DEV)] *= 6.0
    return torch.randn(rows, n, generator=gen, device=DEV, dtype=dt).mul_(channel.to(dt))


def _int8(gen, rows, n):
    """8-bit rows of normally distributed values whose largest lie near four deviations, 16 bytes apart or a multiple, as the
    quantisers lay them out."""
    q = torch.zeros(rows, -(-n // 16) * 16, dtype=torch.int8, device=DEV)
    step = max(1, (1 << 27) // q.shape[1])
    for at in range(0, rows, step):
        part = q[at:at + step, :n]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV).mul_(127.0 / 4.0).round_().clamp_(-127, 127))
    return q[:, :n]


def _scales(gen, n, typical):
    return typical * torch.exp(0.3 * torch.randn(n, generator=gen, device=DEV))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s, kind = {"case": case}, case["kind"]
    if kind in ("gemm8", "project"):
        m, n, k = case["m"], case["n"], case["k"]
        s["b"], s["b_scale"] = _int8(gen, n, k), _scales(gen, n, 0.06 / 127)
        if kind == "gemm8":
            s["a"], s["a_scale"] = _int8(gen, m, k), _scales(gen, m, 4.0 / 127)
            dt = DTYPES[case["out"]]
            s["bias"] = torch.randn(n, generator=gen, device=DEV).to(dt) if case["bias"] else None
            return s
        dt = DTYPES[case["dtype"]]
        s["x"], s["residual"] = torch.randn(m, k, generator=gen, device=DEV, dtype=dt), _hidden(gen, m, k, dt)
        s["w"], s["eps"] = torch.randn(k, generator=gen, device=DEV).mul_(0.2).add_(1.0).to(dt), 1e-6
        return s
    rows, n, dt = case["rows"], case["n"], DTYPES[case["dtype"]]
    s["x"] = _hidden(gen, rows, n, dt)
    if kind == "quant":
        return s
    s["residual"] = _hidden(gen, rows, n, dt) if case["residual"] else None
    s["w"] = torch.randn(n, generator=gen, device=DEV).mul_(0.2).add_(0.0 if case["plus_one"] else 1.0).to(DTYPES[case["wdtype"]])
    s["eps"] = 1e-6
    if kind == "norm_grad":  # x is the sum that the forward pass has left, d_sum the gradient that comes back beside the norm
        s["d_y"] = torch.randn(rows, n, generator=gen, device=DEV, dtype=dt)
        s["d_sum"], s["residual"] = s["residual"], None
        s["rstd"] = torch.rsqrt(s["x"].float().square().mean(-1) + s["eps"])
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _weight(case, s):
    return s["w"].float() + 1.0 if case.get("plus_one") else s["w"].float()


def _norm_plain(case, s):
    x = s["x"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    f = h.float()
    rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + s["eps"])
    return f * rstd * _weight(case, s), h, rstd[:, 0]


def _rows_plain(y):
    """Whole numbers in 32 bits and the scale of each row."""
    scale = y.abs().amax(-1, keepdim=True) / 127.0
    return (y / scale).round(), scale


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        y, h, rstd = _norm_plain(case, s)
        return {"y": y.to(h.dtype), "sum": None if s["residual"] is None else h, "rstd": rstd}
    if kind == "norm_grad":
        xh = s["x"].float() * s["rstd"][:, None]
        d_y = s["d_y"].float()
        g = d_y * _weight(case, s)
        dx = s["rstd"][:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
        if s["d_sum"] is not None:
            dx = dx + s["d_sum"].float()
        return {"dx": dx.to(s["x"].dtype), "dw": (d_y * xh).sum(0).to(s["w"].dtype)}
    if kind == "norm8":
        y, h, _ = _norm_plain(case, s)
        q, scale = _rows_plain(y)
        return {"values": (q * scale).to(torch.bfloat16), "scale": scale[:, 0], "sum": None if s["residual"] is None else h}
    if kind == "quant":
        q, scale = _rows_plain(s["x"].float())
        return {"values": (q * scale).to(torch.bfloat16), "scale": scale[:, 0]}
    if kind == "project":
        y, h, _ = _norm_plain(case, s)
        q, scale = _rows_plain(y)
        return {"c": ((q @ s["b"].float().t()) * scale * s["b_scale"]).to(torch.bfloat16), "sum": h}
    c = (s["a"].float() @ s["b"].float().t()).mul_(s["a_scale"][:, None]).mul_(s["b_scale"])
    if s["bias"] is not None:
        c.add_(s["bias"].float())
    return {"c": c.to(DTYPES[case["out"]])}


# ---------------------------------------------------------------------------------------------------------------- own kernels
def _run_own(s):
    from avelang_b200 import gemm, norm
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        got = norm.rms_norm(s["x"], s["w"], s["eps"], residual=s["residual"], zero_centered=case["plus_one"], return_stats=True)
        return {"y": got[0], "sum": None if s["residual"] is None else got[1], "rstd": got[-1]}
    if kind == "norm_grad":
        dx, dw = norm.rms_norm_backward(s["d_y"], s["x"], s["rstd"], s["w"], d_sum=s["d_sum"], zero_centered=case["plus_one"])
        return {"dx": dx, "dw": dw}
    if kind == "norm8":
        got = norm.rms_norm_int8(s["x"], s["w"], s["eps"], residual=s["residual"], zero_centered=case["plus_one"])
        return {"values": gemm.dequantize_rows_int8(got[0], got[1]), "scale": got[1], "sum": None if s["residual"] is None else got[2]}
    if kind == "quant":
        q, scale = gemm.quantize_rows_int8(s["x"])
        return {"values": gemm.dequantize_rows_int8(q, scale), "scale": scale}
    if kind == "project":
        q, scale, h = norm.rms_norm_int8(s["x"], s["w"], s["eps"], residual=s["residual"])
        return {"c": gemm.gemm_int8_transposed_b(q, s["b"], scale, s["b_scale"]), "sum": h}
    return {"c": gemm.gemm_int8_transposed_b(s["a"], s["b"], s["a_scale"], s["b_scale"], s["bias"], out_dtype=DTYPES[case["out"]])}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    kind, size = case["kind"], {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind in ("gemm8", "project"):
        m, n, k = case["m"], case["n"], case["k"]
        bytes_, flops = n * k + 4 * n, 2 * m * n * k
        if kind == "gemm8":
            return {"bytes": bytes_ + m * k + 4 * m + m * n * size[case["out"]] + (n * size[case["out"]] if case["bias"] else 0), "flops": flops}
        e = size[case["dtype"]]
        return {"bytes": bytes_ + m * k * 3 * e + k * e + m * n * 2, "flops": flops + 8 * m * k}
    rows, n, e = case["rows"], case["n"], size[case["dtype"]]
    if kind == "quant":
        return {"bytes": rows * n * (e + 2) + rows * 4, "flops": 4 * rows * n}
    r, w = (1 if case["residual"] else 0), n * size[case["wdtype"]]
    if kind == "norm":
        return {"bytes": rows * n * e * (2 + 2 * r) + rows * 4 + w, "flops": (5 + r) * rows * n}
    if kind == "norm_grad":
        return {"bytes": rows * n * e * (3 + r) + rows * 4 + 2 * w, "flops": (10 + r) * rows * n}
    return {"bytes": rows * n * (e * (1 + 2 * r) + 2) + rows * 4 + w, "flops": (9 + r) * rows * n}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_norm(x, residual, w, plus_one, eps):
    h = x if residual is None else torch.add(x.double(), residual.double()).to(x.dtype)
    d = h.double()
    mean_square = torch.einsum("rn,rn->r", d, d) / d.shape[1]
    rstd = 1.0 / torch.sqrt(mean_square + eps)
    return torch.einsum("rn,r,n->rn", d, rstd, w.double() + (1.0 if plus_one else 0.0)), h, rstd


def _exact_rows(y):
    top = torch.maximum(y.amax(1), -y.amin(1))
    return torch.round(y * (127.0 / top)[:, None]), top / 127.0


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    with torch.no_grad():
        if kind == "gemm8":
            c = torch.matmul(s["a"].double(), s["b"].double().t())
            c.mul_(s["b_scale"].double()[None]).mul_(s["a_scale"].double()[:, None])
            return {"c": c if s["bias"] is None else c.add_(s["bias"].double()[None])}
        if kind == "quant":
            q, scale = _exact_rows(s["x"].double())
            return {"values": q * scale[:, None], "scale": scale}
        if kind == "norm_grad":
            xh = torch.einsum("rn,r->rn", s["x"].double(), s["rstd"].double())
            d_y = s["d_y"].double()
            g = d_y * (s["w"].double() + (1.0 if case["plus_one"] else 0.0))[None]
            along = torch.einsum("rn,rn->r", g, xh) / xh.shape[1]
            dx = torch.einsum("rn,r->rn", g - along[:, None] * xh, s["rstd"].double())
            return {"dx": dx if s["d_sum"] is None else dx + s["d_sum"].double(), "dw": torch.einsum("rn,rn->n", d_y, xh)}
        y, h, rstd = _exact_norm(s["x"], s["residual"], s["w"], case.get("plus_one", False), s["eps"])
        if kind == "norm":
            return {"y": y, "sum": None if s["residual"] is None else h.double(), "rstd": rstd}
        q, scale = _exact_rows(y)
        if kind == "norm8":
            return {"values": q * scale[:, None], "scale": scale, "sum": None if s["residual"] is None else h.double()}
        c = torch.matmul(q, s["b"].double().t()) * scale[:, None] * s["b_scale"].double()[None]
        return {"c": c, "sum": h.double()}
