"""Linear attention with a decay for each head, and layer norm, as cases that can be timed and whose outputs can be compared.

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t          (S fp32 [dk, dv] of one sequence and value head)
    y = (x - mean) rstd weight + bias                                    (over the last dimension)

Head counts follow the repository's layer (16 key heads, 32 value heads, head dimension 128, hidden size 2048) and its
head-sharded forms; token counts run from one decoded token to a packed batch of 65536.  ``run`` computes each operator in
elementary operations in 32 bits, or, where ``own`` is true, through the framework's entry points.  Inputs are made on the
GPU from the seed alone.
"""
import math
import random

import torch

own = False
DEV = "cuda"
CHUNK = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one user's token: the smallest call, all latency
        {"name": "decode_one", "kind": "decode", "n": 1, "hk": 16, "hv": 32, "dk": 128, "dv": 128, "gate": "token"},
        # the continuous-batching step at its full size: 256 sequences over a pool of 512 slots
        {"name": "decode_pool", "kind": "decode", "n": 256, "hk": 16, "hv": 32, "dk": 128, "dv": 128, "gate": "token"},
        # time to first token of a chat message: one short prompt of odd length that continues from a state
        {"name": "prefill_short", "kind": "prefill", "b": 1, "t": 203, "seqs": 0, "hk": 16, "hv": 32, "dk": 128, "dv": 128,
         "gate": "token", "state": True},
        # a layer's prefill of one 8192-token prompt
        {"name": "prefill_layer", "kind": "prefill", "b": 1, "t": 8192, "seqs": 0, "hk": 16, "hv": 32, "dk": 128, "dv": 128,
         "gate": "token", "state": False},
        # the heads one of eight GPUs owns, on a long document, with one decay a head
        {"name": "prefill_sharded", "kind": "prefill", "b": 1, "t": 32768, "seqs": 0, "hk": 4, "hv": 4, "dk": 128, "dv": 128,
         "gate": "head", "state": False},
        # a packed batch of prompts of very unequal length that continue from states
        {"name": "prefill_packed", "kind": "prefill", "b": 1, "t": 65536, "seqs": 24, "hk": 16, "hv": 32, "dk": 128, "dv": 128,
         "gate": "token", "state": True},
        # a training step of the layer: forward pass and the gradients of every input
        {"name": "train_layer", "kind": "train", "b": 2, "t": 4096, "seqs": 0, "hk": 16, "hv": 32, "dk": 128, "dv": 128,
         "gate": "token", "state": True},
        # a training step on packed documents, value heads of 64 and one decay a head
        {"name": "train_packed", "kind": "train", "b": 1, "t": 3001, "seqs": 5, "hk": 8, "hv": 8, "dk": 128, "dv": 64,
         "gate": "head", "state": False},
        # the norm in front of a decode step's projection
        {"name": "norm_decode", "kind": "norm", "rows": 37, "n": 2048, "dtype": "bf16", "wdtype": "bf16"},
        # the norm in front of the block's projection at its largest
        {"name": "norm_block", "kind": "norm", "rows": 131072, "n": 2048, "dtype": "bf16", "wdtype": "fp32"},
        # the norm's gradients in the training step of the layer
        {"name": "norm_grad", "kind": "norm_grad", "rows": 8192, "n": 2048, "dtype": "bf16", "wdtype": "fp32"},
        # the same in 32 bits at an odd width
        {"name": "norm_grad_odd", "kind": "norm_grad", "rows": 1001, "n": 1409, "dtype": "fp32", "wdtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "packed", "train", "train", "norm", "norm_grad"])
    hk, hv = rng.choice([(2, 4), (4, 4), (8, 8), (8, 16), (16, 32), (32, 32), (1, 8)])
    heads = {"hk": hk, "hv": hv, "dk": rng.choice([64, 128, 128]), "dv": rng.choice([64, 128, 128]), "gate": rng.choice(["token", "token", "head", "none"])}
    if kind == "decode":
        return {"kind": "decode", "n": _log_int(rng, 1, 256), **heads}
    if kind == "prefill":  # one dense prompt or a few
        b = rng.choice([1, 1, 2, 3])
        return {"kind": "prefill", "b": b, "t": _log_int(rng, 33, min(32768, 262144 // hv) // b), "seqs": 0, **heads, "state": rng.random() < 0.5}
    if kind == "packed":
        t = _log_int(rng, 300, min(65536, 2097152 // hv))
        return {"kind": "prefill", "b": 1, "t": t, "seqs": _log_int(rng, 1, min(24, t // 64)), **heads, "state": rng.random() < 0.5}
    if kind == "train":
        packed = rng.random() < 0.3
        b = 1 if packed else rng.choice([1, 2])
        t = _log_int(rng, 65, 4096)
        return {"kind": "train", "b": b, "t": t, "seqs": rng.randint(1, 1 + t // 64) if packed else 0, **heads, "state": rng.random() < 0.5}
    n = rng.choice([64, 1000, 2048, 4096, 8192]) if rng.random() < 0.6 else _log_int(rng, 17, 16384)
    most = 131072 * 2048 // n if kind == "norm" else 32768 * 2048 // n
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return {"kind": kind, "rows": _log_int(rng, 1, min(131072, most // 2 if dt == "fp32" else most)), "n": n, "dtype": dt,
            "wdtype": rng.choice(["fp32", dt])}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    x = torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)
    return x if std == 1.0 else x.mul_(std)


def _gate(gen, case, b, t):
    """Logarithms of the decays: for every token and head, for every head, or none at all."""
    hv = case["hv"]
    if case["gate"] == "none":
        return None
    if case["gate"] == "head":  # a geometric range of reaches, from a few tokens to a few hundred of them
        slope = torch.exp2(-8.0 * (torch.arange(hv, device=DEV) + 1.0) / hv)
        return -slope * (0.9 + 0.2 * torch.rand(hv, generator=gen, device=DEV))
    a_log = torch.rand(hv, generator=gen, device=DEV) * math.log(16.0) - math.log(16.0)
    return -torch.exp(a_log) * torch.nn.functional.softplus(torch.randn(b, t, hv, generator=gen, device=DEV) - 1.0)


def _lengths(seed, n, total):
    """n sequence lengths, log-uniform over two decades before they are scaled to sum to total."""
    rng = random.Random(int(seed) * 7919 + n)
    w = [math.exp(rng.uniform(0.0, math.log(128.0))) for _ in range(n)]
    lens = [max(1, int(x * total / sum(w))) for x in w]
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


def prepare(case, seed):
    gen = _gen(seed)
    s = {"case": case}
    if case["kind"] in ("norm", "norm_grad"):
        dt, wdt, n = DTYPES[case["dtype"]], DTYPES[case["wdtype"]], case["n"]
        s["x"] = _normal(gen, case["rows"], n, dtype=dt).mul_(1.5).add_(0.25)
        s["w"] = _normal(gen, n, dtype=torch.float32).mul_(0.2).add_(1.0).to(wdt)
        s["bias"] = _normal(gen, n, dtype=torch.float32).mul_(0.2).to(wdt)
        s["eps"] = 1e-5
        if case["kind"] == "norm_grad":
            s["dy"] = _normal(gen, case["rows"], n, dtype=dt)
            s["mean"], s["rstd"] = _stats(s["x"], s["eps"])
        return s
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    if case["kind"] == "decode":
        n = case["n"]
        s["q"], s["k"], s["v"] = _normal(gen, n, 1, hk, dk), _normal(gen, n, 1, hk, dk), _normal(gen, n, 1, hv, dv)
        s["g"] = _gate(gen, case, n, 1)
        s["pool"] = _normal(gen, 2 * n, hv, dk, dv, dtype=torch.float32)
        s["idx"] = torch.randperm(2 * n, generator=gen, device=DEV)[:n].to(torch.int32).contiguous()
        return s
    b, t = case["b"], case["t"]
    s["q"], s["k"], s["v"] = _normal(gen, b, t, hk, dk), _normal(gen, b, t, hk, dk), _normal(gen, b, t, hv, dv)
    s["g"] = _gate(gen, case, b, t)
    lens = _lengths(seed, case["seqs"], t) if case["seqs"] else None
    s["cu"] = None
    if lens:
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    n = len(lens) if lens else b
    s["state"] = _normal(gen, n, hv, dk, dv, dtype=torch.float32) if case["state"] else None
    s["plan"] = _plan(lens or [t] * b)
    if case["kind"] == "train":
        s["d_o"] = _normal(gen, b, t, hv, dv)
        s["d_final"] = _normal(gen, n, hv, dk, dv, std=0.1, dtype=torch.float32)
        for name in ("q", "k", "v", "g", "state"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _plan(lens):
    """Chunks of the sequences laid end to end: token indices [M, 64], which of them exist, and the chunks in the order of
    their place in a sequence."""
    index, valid, steps, at = [], [], [], 0
    for n, length in enumerate(lens):
        for j in range(0, length, CHUNK):
            index.append([min(at + j + i, at + length - 1) for i in range(CHUNK)])
            valid.append([j + i < length for i in range(CHUNK)])
            while len(steps) <= j // CHUNK:
                steps.append(([], []))
            steps[j // CHUNK][0].append(n)
            steps[j // CHUNK][1].append(len(index) - 1)
        at += length
    dev = lambda x, dt=torch.long: torch.tensor(x, dtype=dt, device=DEV)
    return {"index": dev(index), "valid": dev(valid, torch.bool), "steps": [(dev(a), dev(c)) for a, c in steps], "n": len(lens)}


def _scan(q, k, v, g, scale, state, plan):
    """The operator over whole sequences in 32 bits, 64 tokens at a time; q, k with as many heads as v."""
    shape, hv, dk, dv = v.shape, v.shape[2], q.shape[3], v.shape[3]
    index, valid = plan["index"], plan["valid"]
    rows = lambda x: x.reshape(-1, *x.shape[2:])[index].transpose(1, 2).float()          # [M, H, 64, d]
    keep = valid[:, None, :, None]
    qc, kc, vc = rows(q), rows(k) * keep, rows(v) * keep
    gc = torch.zeros(len(index), hv, CHUNK, dtype=torch.float64, device=DEV)
    if g is not None:
        per_token = g.expand(shape[0], shape[1], hv) if g.dim() == 1 else g
        gc = per_token.reshape(-1, hv)[index].transpose(1, 2).double() * valid[:, None, :]
    cum = gc.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=DEV).tril()
    decay = torch.where(lower, cum[..., :, None] - cum[..., None, :], -math.inf).exp().float()
    local = (kc * (cum[..., -1:] - cum).exp().float()[..., None]).transpose(-1, -2) @ vc   # [M, H, dk, dv]
    total = cum[..., -1].exp().float()[..., None, None]
    now = torch.zeros(plan["n"], hv, dk, dv, device=DEV) if state is None else state
    order, entering = [], []
    for seqs, chunks in plan["steps"]:
        order.append(chunks)
        entering.append(now[seqs])
        now = now.index_copy(0, seqs, entering[-1] * total[chunks] + local[chunks])
    states = torch.cat(entering)[torch.argsort(torch.cat(order))]
    out = ((qc @ kc.transpose(-1, -2)) * decay) @ vc + (qc @ states) * cum.exp().float()[..., None]
    there = valid.reshape(-1)
    o = torch.zeros(shape[0] * shape[1], hv, dv, device=DEV)
    o = o.index_copy(0, index.reshape(-1)[there], out.transpose(1, 2).reshape(-1, hv, dv)[there])
    return (scale * o).view(shape), now


def _shared(x, hv):
    """Every value head's key head."""
    return x.repeat_interleave(hv // x.shape[2], dim=2)


def _stats(x, eps):
    x = x.float()
    mean = x.mean(-1)
    return mean, ((x - mean[:, None]).square().mean(-1) + eps).rsqrt()


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        mean, rstd = _stats(s["x"], s["eps"])
        y = (s["x"].float() - mean[:, None]) * rstd[:, None] * s["w"].float() + s["bias"].float()
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    if kind == "norm_grad":
        x, dy, rstd = s["x"].float(), s["dy"].float(), s["rstd"][:, None]
        xh = (x - s["mean"][:, None]) * rstd
        wdy = dy * s["w"].float()
        dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True))
        wdt = s["w"].dtype
        return {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0, dtype=torch.float64).to(wdt), "db": dy.sum(0, dtype=torch.float64).to(wdt)}
    scale, hv = case["dk"] ** -0.5, case["hv"]
    if kind == "decode":
        idx = s["idx"].long()
        q, k, v = _shared(s["q"], hv)[:, 0].float(), _shared(s["k"], hv)[:, 0].float(), s["v"][:, 0].float()
        state = s["pool"][idx]
        if s["g"] is not None:
            g = s["g"] if s["g"].dim() == 1 else s["g"][:, 0]
            state = state * g.exp()[..., None, None]
        state = state + k[..., :, None] * v[..., None, :]
        s["pool"][idx] = state
        o = scale * (q[..., None, :] @ state)[..., 0, :]
        return {"o": o[:, None].to(torch.bfloat16), "pool": s["pool"]}
    if kind == "prefill":
        o, final = _scan(_shared(s["q"], hv), _shared(s["k"], hv), s["v"], s["g"], scale, s["state"], s["plan"])
        return {"o": o.to(torch.bfloat16), "final": final}
    wanted = [x for x in (s["q"], s["k"], s["v"], s["g"], s["state"]) if x is not None]
    # 32-bit copies of the inputs: the gradients are rounded once, behind the sum over the value heads of a key head
    wide = {name: None if s[name] is None else s[name].detach().float().requires_grad_(True) for name in ("q", "k", "v", "g", "state")}
    o, final = _scan(_shared(wide["q"], hv), _shared(wide["k"], hv), wide["v"], wide["g"], scale, wide["state"], s["plan"])
    grads = torch.autograd.grad([o, final], [x for x in wide.values() if x is not None], [s["d_o"].float(), s["d_final"]])
    return {"o": o.detach().to(torch.bfloat16), "final": final.detach(), "grads": [d.to(x.dtype) for d, x in zip(grads, wanted)]}


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return _plain(s)
    from avelang_b200 import linear_attention, norm
    case, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        y, mean, rstd = norm.layer_norm(s["x"], s["w"], s["bias"], s["eps"], return_stats=True)
        return {"y": y, "mean": mean, "rstd": rstd}
    if kind == "norm_grad":
        dx, dw, db = norm.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
        return {"dx": dx, "dw": dw, "db": db}
    if kind == "decode":
        o, pool = linear_attention.fused_recurrent_linear_attention(s["q"], s["k"], s["v"], s["g"], initial_state=s["pool"], state_indices=s["idx"])
        return {"o": o, "pool": pool}
    if kind == "prefill":
        o, final = linear_attention.chunk_linear_attention(s["q"], s["k"], s["v"], s["g"], initial_state=s["state"],
                                                           output_final_state=True, cu_seqlens=s["cu"])
        return {"o": o, "final": final}
    o, final = linear_attention.LinearAttentionFunction.apply(s["q"], s["k"], s["v"], s["g"], None, s["state"], s["cu"])
    wanted = [x for x in (s["q"], s["k"], s["v"], s["g"], s["state"]) if x is not None]
    grads = torch.autograd.grad([o, final], wanted, [s["d_o"], s["d_final"]])
    return {"o": o.detach(), "final": final.detach(), "grads": list(grads)}


# ---------------------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _recurrence(q, k, v, g, scale, state, lens, heads_g):
    """Token by token, the sequences side by side, the longest first; returns o and the final states."""
    running = sorted(range(len(lens)), key=lambda n: -lens[n])
    order = torch.tensor(running, device=DEV)
    starts = torch.tensor([sum(lens[:n]) for n in running], device=DEV)
    o = torch.zeros(v.shape[0], v.shape[1], v.shape[2], dtype=torch.float64, device=DEV)
    now, count = state[order], len(running)
    for t in range(max(lens)):
        while lens[running[count - 1]] <= t:
            count -= 1
        tok, part = starts[:count] + t, now[:count]
        if g is not None:
            part.mul_(torch.exp(g[tok] if not heads_g else g[None])[..., None, None])
        part.addcmul_(k[tok][..., :, None], v[tok][..., None, :])
        o[tok] = scale * torch.matmul(q[tok][..., None, :], part)[..., 0, :]
    final = torch.empty_like(now)
    final[order] = now
    return o, final


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        x, w = s["x"].double(), s["w"].double()
        if kind == "norm":
            mean, var = x.mean(-1), x.var(-1, unbiased=False)
            rstd = 1.0 / torch.sqrt(var + s["eps"])
            return {"y": (x - mean[:, None]) * rstd[:, None] * w + s["bias"].double(), "mean": mean, "rstd": rstd}
        dy, xh = s["dy"].double(), (x - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        n, inner = case["n"], dy * w
        dx = (n * inner - inner.sum(-1, keepdim=True) - xh * (inner * xh).sum(-1, keepdim=True)) * (s["rstd"].double()[:, None] / n)
        return {"dx": dx, "dw": torch.einsum("rn,rn->n", dy, xh), "db": dy.sum(0)}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    group = torch.arange(hv, device=DEV) // (hv // hk)
    flat = lambda x: x.detach().double().flatten(0, 1)
    q, k, v = flat(s["q"])[:, group], flat(s["k"])[:, group], flat(s["v"])
    heads_g = case["gate"] == "head"
    g = None if s["g"] is None else s["g"].detach().double() if heads_g else flat(s["g"])
    scale = dk ** -0.5
    if kind == "decode":
        n, idx = case["n"], s["idx"].long()
        o, final = _recurrence(q, k, v, g, scale, s["pool"][idx].double(), [1] * n, heads_g)
        pool = s["pool"].double()
        pool[idx] = final
        return {"o": o[:, None], "pool": pool}
    cu = s["cu"].tolist() if s["cu"] is not None else [i * case["t"] for i in range(case["b"] + 1)]
    lens = [e - a for a, e in zip(cu, cu[1:])]
    n, longest = len(lens), max(lens)
    if longest > 40000:  # a step a token
        return None
    state = torch.zeros(n, hv, dk, dv, dtype=torch.float64, device=DEV) if s["state"] is None else s["state"].detach().double()
    o, final = _recurrence(q, k, v, g, scale, state, lens, heads_g)
    shape = s["v"].shape
    if kind == "prefill":
        return {"o": o.view(shape), "final": final}
    # The gradients are recurrences of the same form: dq_t = scale S_t do_t forwards, dk_t = R_t v_t and dv_t = R_t^T k_t backwards in
    # time with R_t = scale q_t do_t^T + exp(g_{t+1}) R_{t+1}; and g_t has the gradient sum_{s >= t} (q_s.dq_s - k_s.dk_s) + <S_T, R_T>.
    d_o, d_final = flat(s["d_o"]), s["d_final"].double()
    back = torch.cat([torch.arange(e - 1, a - 1, -1) for a, e in zip(cu, cu[1:])]).to(DEV)   # its own inverse
    tokens = q.shape[0]
    per_token = None if g is None else g[None].expand(tokens, hv) if heads_g else g
    shifted = None
    if g is not None:
        shifted = torch.zeros(tokens, hv, dtype=torch.float64, device=DEV)
        shifted[:-1] = per_token[1:]
        shifted[torch.tensor([e - 1 for e in cu[1:]], device=DEV)] = 0.0
        shifted = shifted[back]
    dq, _ = _recurrence(d_o, v, k, g, scale, state.transpose(-1, -2), lens, heads_g)
    kb, vb, qb, ob = k[back], v[back], q[back] * scale, d_o[back]
    dk_, _ = _recurrence(vb, ob, qb, shifted, 1.0, d_final.transpose(-1, -2), lens, False)
    dv_, last = _recurrence(kb, qb, ob, shifted, 1.0, d_final, lens, False)
    dk_, dv_ = dk_[back], dv_[back]
    grads = [x.view(tokens, hk, hv // hk, dk).sum(2).view(s["q"].shape) for x in (dq, dk_)] + [dv_.view(shape)]
    if g is not None:
        dg = torch.empty(tokens, hv, dtype=torch.float64, device=DEV)
        term, ends = (q * dq - k * dk_).sum(-1), (final * d_final).sum((-1, -2))
        for i, (a, e) in enumerate(zip(cu, cu[1:])):
            dg[a:e] = term[a:e].flip(0).cumsum(0).flip(0) + ends[i]
        grads.append(dg.sum(0) if heads_g else dg.view(s["g"].shape))
    if s["state"] is not None:
        first = torch.tensor(cu[:-1], device=DEV)
        grads.append(last if g is None else last * torch.exp(per_token[first])[..., None, None])
    return {"o": o.view(shape), "final": final, "grads": grads}


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        size, wsize = DTYPES[case["dtype"]].itemsize, DTYPES[case["wdtype"]].itemsize
        cells, rows, n = case["rows"] * case["n"], case["rows"], case["n"]
        if kind == "norm":
            return {"bytes": 2.0 * cells * size + 2 * n * wsize + 8 * rows, "flops": 8.0 * cells}
        return {"bytes": 3.0 * cells * size + 3 * n * wsize + 8 * rows, "flops": 14.0 * cells}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    state = 4.0 * hv * dk * dv
    gate = 4.0 * hv if case["gate"] == "token" else 0.0
    if kind == "decode":
        n = case["n"]
        return {"bytes": n * (2 * state + 4.0 * hk * dk + 4.0 * hv * dv + gate), "flops": n * hv * 5.0 * dk * dv}
    tokens, n = case["b"] * case["t"], case["seqs"] or case["b"]
    # in chunks of 64 tokens: half of Q K^T (once a key head) and of P V, Q S and K^T V
    flops = tokens * (hk * 64.0 * dk + hv * (64.0 * dv + 4.0 * dk * dv))
    forward = tokens * (4.0 * hk * dk + 4.0 * hv * dv + gate) + n * state * (2 if case["state"] else 1)
    if kind == "prefill":
        return {"bytes": forward, "flops": flops}
    # the gradients read q, k, v, g, do and the states, and write dq, dk, dv, dg and the states'
    backward = tokens * (8.0 * hk * dk + 6.0 * hv * dv + 2 * gate) + n * state * (3 if case["state"] else 1)
    return {"bytes": forward + backward, "flops": 4.0 * flops}
