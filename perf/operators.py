"""The training operators of a transformer layer (attention, layer norm, Linear with its epilogue): cases, plain forms, exact values.

`run` computes a case with elementary torch operations in 32 bits, or -- where `own` is true -- through `HipEngine`'s operators.  Batches
are what the simulator trains on: scenes of agents, map polylines and their nodes, most of them padded, plus the generic sizes of the
same operators (wider features, longer sequences, shared key / value heads)."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_engines = {}


def _engine():
    """The engine a user's program holds (one per process)."""
    from trafficbots_amd.config import load_model_config
    from trafficbots_amd.runtime import HipEngine

    if "engine" not in _engines:
        _engines["engine"] = HipEngine(load_model_config())
    return _engines["engine"]


# ------------------------------------------------------------------------------------------------- cases
def _attention(name, b, lq, lk, h, hkv, d, dtype, train, causal=False, eye=False, padded=True):
    return {"name": name, "op": "attention", "b": b, "lq": lq, "lk": lk, "h": h, "hkv": hkv, "d": d, "dtype": dtype, "train": train,
            "causal": causal, "eye": eye, "padded": padded}


def _layer_norm(name, rows, c, dtype):
    return {"name": name, "op": "layer_norm", "rows": rows, "c": c, "dtype": dtype}


def _linear(name, m, k, n, dtype, backward, relu, residual, padded):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "backward": backward, "relu": relu,
            "residual": residual, "padded": padded}


def listed():
    return [
        # one agent asks a long map: a single query row, forward only (closed-loop serving; latency)
        _attention("one agent, map", 1, 1, 1024, 4, 4, 32, "fp32", False),
        # 32 scenes of 64 agents against 256 polylines, the headline batch of a training step
        _attention("agents to map", 32, 64, 256, 4, 4, 32, "fp32", True),
        # the 20 nodes of every polyline attend to each other: 8192 tiny problems
        _attention("polyline nodes", 8192, 20, 20, 4, 4, 32, "fp32", True),
        # polylines attend to each other in the real map size
        _attention("map to map", 32, 1024, 1024, 4, 4, 32, "bf16", True),
        # agents attend to each other but not to themselves; odd sizes, some rows have nobody to look at
        _attention("agents to agents", 33, 61, 61, 4, 4, 32, "bf16", True, eye=True),
        # a long causal sequence with shared key / value heads
        _attention("long causal", 1, 8192, 8192, 16, 4, 128, "bf16", True, causal=True, padded=False),
        # layer norm of the agents of a batch (latency)
        _layer_norm("norm of agents", 2048, 128, "fp32"),
        # layer norm of all map nodes of a batch at the real map size
        _layer_norm("norm of nodes", 655360, 128, "bf16"),
        # wide odd rows
        _layer_norm("norm of wide rows", 8191, 2047, "fp32"),
        # the attribute encoder's first Linear: eleven inputs
        _linear("agent attributes", 704, 11, 32, "fp32", False, True, False, True),
        # the feed-forward's first Linear over all map nodes, backward
        _linear("feed-forward of nodes", 163840, 128, 128, "fp32", True, True, False, True),
        # a wide projection that adds its residual
        _linear("wide projection", 16384, 2048, 2048, "bf16", False, False, True, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "layer_norm", "linear"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "attention":
        hkv = rng.choice([1, 2, 4])
        h = hkv * rng.choice([1, 1, 2, 4])
        d = 8 * rng.randint(1, 16)
        lq, lk = _log(rng, 1, 4096), _log(rng, 1, 4096)
        causal = rng.random() < 0.3
        if rng.random() < 0.5:
            lk = lq
        train = rng.random() < 0.7
        if train:  # with a handful of keys the scores' gradients are all rounding
            lk = max(lk, 8)
        most = max(1, min(8192, (1 << 27) // (h * lq * lk), (1 << 25) // (max(lq, lk) * h * d)))
        eye = not causal and lq == lk and lk >= 8 and rng.random() < 0.3
        c = _attention("", _log(rng, 1, most), lq, lk, h, hkv, d, dtype, train, causal, eye, rng.random() < 0.6)
    elif op == "layer_norm":
        width = _log(rng, 8, 8192)
        c = _layer_norm("", _log(rng, 1, min(655360, (1 << 26) // width)), width, dtype)
    else:
        k, n = _log(rng, 8, 2048), _log(rng, 8, 2048)
        most = min(655360, (1 << 26) // max(k, n), (1 << 35) // (k * n))
        c = _linear("", _log(rng, 1, most), k, n, dtype, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(t)

    def valid(*shape):
        return torch.rand(*shape, device="cuda", generator=g) < 0.8

    s = {"case": case}
    if case["op"] == "attention":
        b, lq, lk, h, hkv, d = (case[x] for x in ("b", "lq", "lk", "h", "hkv", "d"))
        s["q"] = normal(b, lq, h, d)
        # keys and values lie side by side, as one projection writes them
        kv = normal(b, lk, 2, hkv, d)
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["query_valid"] = valid(b, lq) if case["padded"] else None
        s["key_valid"] = valid(b, lk) if case["padded"] else None
        if case["padded"]:
            s["key_valid"][: b // 8] = False  # scenes in which nothing can be seen
            s["key_valid"][-1, :8] = s["query_valid"][-1, -1] = True
        s["attn_mask"] = torch.eye(lq, dtype=torch.bool, device="cuda") if case["eye"] else None
        s["d_out"] = normal(b, lq, h, d) if case["train"] else None
    elif case["op"] == "layer_norm":
        rows, c = case["rows"], case["c"]
        s["x"] = (torch.randn(rows, c, device="cuda", generator=g) * 1.5 + torch.randn(rows, 1, device="cuda", generator=g)).to(t)
        s["weight"] = (1.0 + 0.1 * torch.randn(c, device="cuda", generator=g)).to(t)
        s["bias"] = normal(c, scale=0.1)
        s["d_out"] = normal(rows, c)
    else:
        m, k, n = case["m"], case["k"], case["n"]
        s["x"], s["weight"] = normal(m, k), normal(n, k, scale=1.0 / math.sqrt(k))
        s["bias"] = normal(n, scale=0.1)
        s["row_valid"] = valid(m) if case["padded"] else None
        if case["backward"]:
            s["d_out"] = normal(m, n)
            # what the forward pass of the same step kept for the activation's gradient
            s["act"] = normal(m, n).clamp_min_(0) if case["relu"] else None
        else:
            s["residual"] = normal(m, n) if case["residual"] else None
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    return {"attention": _run_attention, "layer_norm": _run_layer_norm, "linear": _run_linear}[s["case"]["op"]](s)


def _run_attention(s):
    case = s["case"]
    if own:
        e = _engine()
        masks = {"query_valid": s["query_valid"], "key_valid": s["key_valid"], "attn_mask": s["attn_mask"], "causal": case["causal"]}
        out, lse = e.attention(s["q"], s["k"], s["v"], **masks)
        if not case["train"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = e.attention_backward(s["d_out"], s["q"], s["k"], s["v"], out, lse, **masks)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    b, lq, lk, h, hkv, d = (case[x] for x in ("b", "lq", "lk", "h", "hkv", "d"))
    t = s["q"].dtype
    scale = 1.0 / math.sqrt(d)
    # [b, hkv, group, l, d]
    q = s["q"].float().view(b, lq, hkv, h // hkv, d).permute(0, 2, 3, 1, 4)
    k = s["k"].float().permute(0, 2, 1, 3).unsqueeze(2)
    v = s["v"].float().permute(0, 2, 1, 3).unsqueeze(2)
    hidden = _hidden(s, lq, lk)
    x = torch.matmul(q * scale, k.transpose(-1, -2))
    if hidden is not None:
        x.masked_fill_(hidden, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = torch.matmul(p, v)
    r = {"out": out.permute(0, 3, 1, 2, 4).reshape(b, lq, h, d).to(t), "lse": lse.reshape(b, h, lq)}
    if case["train"]:
        g = s["d_out"].float().view(b, lq, hkv, h // hkv, d).permute(0, 2, 3, 1, 4)
        dp = torch.matmul(g, v.transpose(-1, -2))
        dv = torch.matmul(p.transpose(-1, -2), g).sum(2)
        ds = dp.sub_((g * out).sum(-1, keepdim=True)).mul_(p)
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(-1, -2), q).sum(2) * scale
        r["dq"] = dq.permute(0, 3, 1, 2, 4).reshape(b, lq, h, d).to(t)
        r["dk"], r["dv"] = dk.permute(0, 2, 1, 3).to(t).contiguous(), dv.permute(0, 2, 1, 3).to(t).contiguous()
    return r


def _hidden(s, lq, lk):
    """True where a query may not see a key, broadcast over [b, hkv, group, lq, lk]; None if everybody sees everything."""
    hidden = None
    if s["key_valid"] is not None:
        hidden = ~(s["query_valid"][:, :, None] & s["key_valid"][:, None, :])[:, None, None]
    if s["attn_mask"] is not None:
        hidden = s["attn_mask"] if hidden is None else hidden | s["attn_mask"]
    if s["case"]["causal"]:
        i = torch.arange(lq, device="cuda")[:, None] + (lk - lq)
        later = torch.arange(lk, device="cuda")[None, :] > i
        hidden = later if hidden is None else hidden | later
    return hidden


def _run_layer_norm(s):
    if own:
        e = _engine()
        y, mean, rstd = e.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
        dx, dw, db = e.layer_norm_backward(s["d_out"], s["x"], s["weight"], mean, rstd)
        return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dw": dw, "db": db}
    t = s["x"].dtype
    x, w, g = s["x"].float(), s["weight"].float(), s["d_out"].float()
    mean = x.mean(-1, keepdim=True)
    x = x - mean
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    x = x * rstd
    y = x * w + s["bias"].float()
    a = g * w
    dx = rstd * (a - a.mean(-1, keepdim=True) - x * (a * x).mean(-1, keepdim=True))
    return {"y": y.to(t), "mean": mean.squeeze(-1), "rstd": rstd.squeeze(-1), "dx": dx.to(t), "dw": (g * x).sum(0).to(t), "db": g.sum(0).to(t)}


def _run_linear(s):
    case = s["case"]
    if own:
        e = _engine()
        if case["backward"]:
            dx, dw, db = e.linear_backward(s["d_out"], s["x"], s["weight"], act=s["act"], row_valid=s["row_valid"])
            return {"dx": dx, "dw": dw, "db": db}
        return {"y": e.linear(s["x"], s["weight"], s["bias"], activation="relu" if case["relu"] else None, row_valid=s["row_valid"],
                              residual=s["residual"])}
    t = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    if case["backward"]:
        dz = s["d_out"].float()
        if s["act"] is not None:
            dz = dz * (s["act"] > 0)
        if s["row_valid"] is not None:
            dz = dz * s["row_valid"][:, None]
        return {"dx": torch.matmul(dz, w).to(t), "dw": torch.matmul(dz.t(), x).to(t), "db": dz.sum(0).to(t)}
    y = torch.matmul(x, w.t()) + s["bias"].float()
    if case["relu"]:
        y = y.clamp_min(0)
    if s["row_valid"] is not None:
        y = y * s["row_valid"][:, None]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(t)}


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        b, lq, lk, h, hkv, d = (case[x] for x in ("b", "lq", "lk", "h", "hkv", "d"))
        pairs = b * h * lq * lk
        if case["causal"]:
            pairs = b * h * sum(max(0, min(lk, i + 1 + lk - lq)) for i in range(lq))
        rows, keys = b * lq * h * d * e, b * lk * hkv * d * e
        masks = (b * (lq + lk) if case["padded"] else 0) + (lq * lk if case["eye"] else 0)
        nbytes, flops = 2 * rows + 2 * keys + 4 * b * h * lq + masks, 4 * d * pairs
        if case["train"]:
            nbytes, flops = nbytes + 2 * rows + 2 * keys, flops + 10 * d * pairs
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "layer_norm":
        rows, c = case["rows"], case["c"]
        return {"bytes": 4 * rows * c * e + 8 * rows + 4 * c * e, "flops": 20 * rows * c}
    m, k, n = case["m"], case["k"], case["n"]
    nbytes = m * k + k * n + n + m * n + (m // e if case["padded"] else 0)
    if case["backward"]:
        return {"bytes": e * (nbytes + m * k + k * n + (m * n if case["relu"] else 0)), "flops": 4 * m * n * k}
    return {"bytes": e * (nbytes + (m * n if case["residual"] else 0)), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "attention":
        return (_exact_layer_norm if case["op"] == "layer_norm" else _exact_linear)(case, s)
    b, lq, lk, h, hkv, d = (case[x] for x in ("b", "lq", "lk", "h", "hkv", "d"))
    f64, dev = torch.float64, "cuda"
    r = {"out": torch.zeros(b, lq, h, d, dtype=f64, device=dev), "lse": torch.full((b, h, lq), -math.inf, dtype=f64, device=dev)}
    if case["train"]:
        r["dq"] = torch.zeros(b, lq, h, d, dtype=f64, device=dev)
        r["dk"], r["dv"] = (torch.zeros(b, lk, hkv, d, dtype=f64, device=dev) for _ in range(2))
    some = max(1, (1 << 27) // (lq * lk))  # scenes a slice: the scores of one head at a time
    for b0 in range(0, b, some):
        z = slice(b0, min(b, b0 + some))
        see = torch.ones(z.stop - z.start, lq, lk, dtype=torch.bool, device=dev)
        if case["causal"]:
            see &= torch.ones(lq, lk, dtype=torch.bool, device=dev).tril(lk - lq)
        if s["attn_mask"] is not None:
            see &= ~s["attn_mask"]
        if s["key_valid"] is not None:
            see &= s["query_valid"][z, :, None]
            see &= s["key_valid"][z, None, :]
        for i in range(h):
            j = i // (h // hkv)
            q, k, v = s["q"][z, :, i].to(f64), s["k"][z, :, j].to(f64), s["v"][z, :, j].to(f64)
            score = torch.where(see, torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d), -math.inf)
            lse = torch.logsumexp(score, -1)
            prob = torch.where(see, torch.exp(score - lse[..., None]), 0.0)
            del score
            out = torch.bmm(prob, v)
            r["out"][z, :, i], r["lse"][z, i] = out, lse
            if case["train"]:
                g = s["d_out"][z, :, i].to(f64)
                r["dv"][z, :, j] += torch.bmm(prob.transpose(1, 2).contiguous(), g)
                change = prob * (torch.bmm(g, v.transpose(1, 2).contiguous()) - (g * out).sum(-1, keepdim=True)) / math.sqrt(d)
                r["dq"][z, :, i] = torch.bmm(change, k)
                r["dk"][z, :, j] += torch.bmm(change.transpose(1, 2).contiguous(), q)
    return r


def _exact_layer_norm(case, s):
    x, w, b, g = (s[i].to(torch.float64) for i in ("x", "weight", "bias", "d_out"))
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    rstd = (var + 1e-5) ** -0.5
    h = (x - mean) * rstd
    c = x.shape[-1]
    dot, flat = torch.mv(g * h, w)[:, None] / c, torch.mv(g, w)[:, None] / c
    return {"y": torch.addcmul(b, h, w), "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": (g * w - flat - h * dot) * rstd,
            "dw": (g * h).sum(0), "db": g.sum(0)}


def _exact_linear(case, s):
    x, w = s["x"].to(torch.float64), s["weight"].to(torch.float64)
    gone = None if s["row_valid"] is None else (~s["row_valid"])[:, None]
    if case["backward"]:
        dz = s["d_out"].to(torch.float64)
        if case["relu"]:
            dz = torch.where(s["act"] > 0, dz, 0.0)
        if gone is not None:
            dz = dz.masked_fill(gone, 0.0)
        return {"dx": torch.mm(dz, w), "dw": torch.mm(dz.t().contiguous(), x), "db": torch.mv(dz.t(), torch.ones(dz.shape[0], dtype=dz.dtype, device=dz.device))}
    y = torch.addmm(s["bias"].to(torch.float64), x, w.t())
    if case["relu"]:
        y = torch.where(y > 0, y, 0.0)
    if gone is not None:
        y = y.masked_fill(gone, 0.0)
    return {"y": y if s["residual"] is None else y + s["residual"].to(torch.float64)}
