"""Measured cases of the operators for distilling and fine-tuning an encoder: attention with its
backward pass, LayerNorm with its backward pass, per-token log probabilities, and the distillation
loss with its gradient.

`run` computes each operator either in plain torch (elementary operations in 32 bits, rounded once
at the end) or, where `own` is true, through the entry points of esm_b200.Model. `exact` gives the
same values from the definitions in 64 bits. Everything is made on the GPU from a seed.
"""
from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases ----------------------------------------------------------------------------------------

def listed():
    return [
        # One protein of 126 residues through the 8M model: a call that is all latency.
        _attn("attention backward 8M 1x128", "backward", "bf16", 20, 16, 1, 128, 128),
        # A right-padded batch of the 35M model, lengths 64 to 512, one entry of it empty.
        _attn("attention backward 35M ragged", "backward", "f16", 20, 24, 32, 64, 512, True),
        # A share of the headline batch of the 650M model, forward and backward.
        _attn("attention forward 650M 16x1024", "forward", "bf16", 20, 64, 16, 1024, 1024),
        _attn("attention backward 650M 16x1024", "backward", "f16", 20, 64, 16, 1024, 1024),
        # Long chains through the 3B model.
        _attn("attention backward 3B 2x4096", "backward", "bf16", 40, 64, 2, 4096, 4096),
        # One masked variant of a 300-residue protein through the 150M model.
        _ln("layernorm backward 150M 302", "backward", "f32", "f16", 302, 640, True),
        # The residual stream of the headline batch: fp32 in, fp16 out, as the encoder has it.
        _ln("layernorm forward 650M 65536", "forward", "f32", "f16", 65536, 1280, False),
        _ln("layernorm backward 650M 65536", "backward", "f32", "f16", 65536, 1280, True),
        # Every token of a mutational scan (300 variants of 302 tokens) scored over the 33 tokens.
        _score("logprobs scan 90600x33", "f32", 90600, 33, 5),
        # A vocabulary of byte-pair or k-mer tokens.
        _score("logprobs 512x32768", "bf16", 512, 32768, 20),
        # A distillation step on the headline batch: all 33 tokens in reach, half of them kept.
        _distill("distillation 65536x33", "f32", 65536, 33, 16, 2.0),
        _distill("distillation 1021x32003", "f16", 1021, 32003, 32, 1.0),
    ]


def _attn(name, way, kind, heads, head_dim, batch, min_len, max_len, empty=False):
    return {"name": name, "op": "attention", "way": way, "type": kind, "heads": heads, "head_dim": head_dim,
            "batch": batch, "min_len": min_len, "max_len": max_len, "empty": empty}


def _ln(name, way, x_type, y_type, rows, dim, residual):
    return {"name": name, "op": "layernorm", "way": way, "x_type": x_type, "y_type": y_type, "rows": rows, "dim": dim,
            "residual": residual}


def _score(name, kind, rows, vocab, k):
    return {"name": name, "op": "logprobs", "type": kind, "rows": rows, "vocab": vocab, "k": k}


def _distill(name, kind, rows, vocab, k, temperature):
    return {"name": name, "op": "distill", "type": kind, "rows": rows, "vocab": vocab, "k": k,
            "temperature": temperature}


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "layernorm", "logprobs", "distill"])
    if op == "attention":
        kind, way = rng.choice(["f16", "bf16"]), rng.choice(["forward", "backward", "backward"])
        heads, head_dim = rng.choice([(20, 16), (20, 24), (20, 32), (20, 64), (40, 64), (rng.randint(1, 16), 8 * rng.randint(1, 8))])
        max_len = _log_uniform(rng, 1, 4096)
        min_len = rng.randint(1, max_len)
        most = max(1, min(64, 2 * 40 * 4096 ** 2 // (heads * max_len ** 2), 65536 // max_len))
        case = _attn("", way, kind, heads, head_dim, _log_uniform(rng, 1, most), min_len, max_len, rng.random() < 0.3)
    elif op == "layernorm":
        dim = rng.choice([320, 480, 640, 1280, 2560, _log_uniform(rng, 16, 8192)])
        rows = _log_uniform(rng, 1, 65536 * 1280 // dim)
        way = rng.choice(["forward", "backward"])
        x_type, y_type = rng.choice(["f32", "f32", "f16", "bf16"]), rng.choice(["f32", "f16", "bf16"])
        case = _ln("", way, x_type, y_type, rows, dim, way == "backward" and rng.random() < 0.5)
    else:
        vocab = rng.choice([33, 33, _log_uniform(rng, 4, 65536)])
        rows = _log_uniform(rng, 1, min(90600, 512 * 32768 // vocab))
        kind, k = rng.choice(["f32", "f16", "bf16"]), rng.randint(1, min(vocab, 48))
        if op == "logprobs":
            case = _score("", kind, rows, vocab, k)
        else:
            case = _distill("", kind, rows, vocab, k, rng.choice([1.0, 2.0, 4.0, 0.5]))
    del case["name"]
    return case


def _lengths(case):
    """Lengths spread over [min_len, max_len] (the last one max_len); the second entry of a batch is empty where asked."""
    lo, hi, n = case["min_len"], case["max_len"], case["batch"]
    lens = [lo + round((hi - lo) * ((i + 1) * 0.6180339887 % 1.0)) for i in range(n - 1)] + [hi]
    if case["empty"] and n > 2:
        lens[1] = 0
    return lens


def work(case):
    if case["op"] == "attention":
        lens, e = _lengths(case), SIZE[case["type"]]
        tokens, d = sum(lens), case["heads"] * case["head_dim"]
        pairs = sum(n * n for n in lens)
        if case["way"] == "forward":
            return {"bytes": 4 * tokens * d * e + 4 * tokens * case["heads"], "flops": 4 * pairs * d}
        return {"bytes": 8 * tokens * d * e + 4 * tokens * case["heads"], "flops": 10 * pairs * d}
    if case["op"] == "layernorm":
        n, ex, ey = case["rows"] * case["dim"], SIZE[case["x_type"]], SIZE[case["y_type"]]
        if case["way"] == "forward":
            return {"bytes": n * (ex + ey) + 8 * case["rows"] + 8 * case["dim"], "flops": 8 * n}
        return {"bytes": n * (2 * ex + ey + (ex if case["residual"] else 0)) + 8 * case["rows"] + 12 * case["dim"],
                "flops": 14 * n}
    n, e, rows, k = case["rows"] * case["vocab"], SIZE[case["type"]], case["rows"], case["k"]
    if case["op"] == "logprobs":
        return {"bytes": n * e + rows * (12 + 8 * k), "flops": 6 * n}
    return {"bytes": 2 * n * e + rows * (12 + 8 * k), "flops": 8 * n}


# ---- inputs ---------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": _prepare_attention, "layernorm": _prepare_layernorm, "logprobs": _prepare_logprobs,
            "distill": _prepare_distill}[case["op"]](case, g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_attention(case, g):
    lens, kind = _lengths(case), TYPES[case["type"]]
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    tokens, H, dh = sum(lens), case["heads"], case["head_dim"]
    # Queries and keys whose scores have a standard deviation of about 1.5, a few heads sharper.
    qkv = _randn(g, tokens, 3, H, dh)
    qkv[:, 0] *= 1.5 * (1.0 + (torch.arange(H, device="cuda") % 5 == 4).float())[:, None]
    s = {"case": case, "qkv": qkv.reshape(tokens, 3 * H * dh).to(kind), "cu": cu, "tokens": tokens,
         "out": torch.empty(tokens, H * dh, dtype=kind, device="cuda"),
         "lse": torch.empty(H, tokens, dtype=torch.float32, device="cuda")}
    if case["way"] == "backward":
        # Gradients of a loss that is scaled for 16-bit training.
        s["dout"] = (0.05 * _randn(g, tokens, H * dh)).to(kind)
        s["dqkv"] = torch.empty_like(s["qkv"])
        s["out"], s["lse"] = _attention_plain(s)
        s["workspace"] = torch.empty(8 * (H * tokens + H * (tokens // 64 + case["batch"] + 1)) + 4096,
                                     dtype=torch.uint8, device="cuda")
    return s


def _prepare_layernorm(case, g):
    n, d, xt, yt = case["rows"], case["dim"], TYPES[case["x_type"]], TYPES[case["y_type"]]
    # A residual stream: a few channels are far larger than the rest, and the rows have an offset.
    x = _randn(g, n, d) * (1.0 + 30.0 * (torch.arange(d, device="cuda") % 211 == 7).float()) + 0.5 * _randn(g, n, 1)
    s = {"case": case, "x": x.to(xt), "w": 1.0 + 0.2 * _randn(g, d), "b": 0.1 * _randn(g, d),
         "mean": torch.empty(n, device="cuda"), "rstd": torch.empty(n, device="cuda")}
    if case["way"] == "forward":
        s["y"] = torch.empty(n, d, dtype=yt, device="cuda")
        return s
    _, s["mean"], s["rstd"] = _layernorm_plain(s["x"], s["w"], s["b"], yt)
    s["dy"] = (0.05 * _randn(g, n, d)).to(yt)
    s["dres"] = (0.05 * _randn(g, n, d)).to(xt) if case["residual"] else None
    s["dx"] = torch.empty_like(s["x"])
    s["dw"], s["db"] = torch.empty_like(s["w"]), torch.empty_like(s["w"])
    s["workspace"] = torch.empty(8 * 1184 * d, dtype=torch.uint8, device="cuda")
    return s


def _logits(case, g):
    """Logits with a spread of 3 around a peak, in reach of each other's rounding so that ties occur."""
    x = 3.0 * _randn(g, case["rows"], case["vocab"]) + 2.0 * _randn(g, case["rows"], 1)
    return x.to(TYPES[case["type"]])


def _prepare_logprobs(case, g):
    n, V, k = case["rows"], case["vocab"], case["k"]
    x = _logits(case, g)
    # Special tokens that a sampler rules out: the first one, and every 97th.
    if V > 8:
        x[:, ::97] = -math.inf
    return {"case": case, "logits": x, "targets": torch.randint(0, V, (n,), generator=g, device="cuda").to(torch.int32),
            "logp": torch.empty(n, device="cuda"), "entropy": torch.empty(n, device="cuda"),
            "top_ids": torch.empty(n, k, dtype=torch.int32, device="cuda"), "top_logp": torch.empty(n, k, device="cuda")}


def _prepare_distill(case, g):
    n, V, k = case["rows"], case["vocab"], case["k"]
    student = _logits(case, g)
    teacher = student.float() + 1.5 * _randn(g, n, V)
    top, ids = teacher.topk(k, dim=1)
    ids = ids.to(torch.int32)
    # Rows with fewer alternatives than k, and a tenth of the tokens without weight (padding).
    short = torch.rand(n, generator=g, device="cuda") < 0.2
    ids[short[:, None] & (torch.arange(k, device="cuda") >= (k + 1) // 2)[None]] = -1
    dloss = torch.rand(n, generator=g, device="cuda") * (torch.rand(n, generator=g, device="cuda") > 0.1)
    return {"case": case, "logits": student, "top_ids": ids, "top_logits": top.contiguous(), "dloss": dloss,
            "loss": torch.empty(n, device="cuda"), "lse": torch.empty(n, device="cuda"),
            "dlogits": torch.empty_like(student)}


# ---- one pass -------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _model():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "codon-infer_b200"))
    import esm_b200

    return esm_b200.Model(0)


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case, _model(), torch.cuda.current_stream().cuda_stream)
    if case["op"] == "attention":
        if case["way"] == "forward":
            out, lse = _attention_plain(state)
            return {"out": out, "lse": lse}
        return {"dqkv": _attention_backward_plain(state)}
    if case["op"] == "layernorm":
        if case["way"] == "forward":
            y, mean, rstd = _layernorm_plain(state["x"], state["w"], state["b"], state["y"].dtype)
            return {"y": y, "mean": mean, "rstd": rstd}
        return _layernorm_backward_plain(state)
    if case["op"] == "logprobs":
        return _logprobs_plain(state)
    return _distill_plain(state)


def _run_own(s, case, m, stream):
    if case["op"] == "attention":
        if case["way"] == "forward":
            m.attention(s["qkv"], s["cu"], case["max_len"], case["heads"], s["out"], s["lse"], stream=stream)
            return {"out": s["out"], "lse": s["lse"]}
        m.attention_backward(s["qkv"], s["cu"], case["max_len"], case["heads"], s["out"], s["lse"], s["dout"],
                             s["dqkv"], s["workspace"], stream=stream)
        return {"dqkv": s["dqkv"]}
    if case["op"] == "layernorm":
        if case["way"] == "forward":
            m.layernorm(s["x"], s["w"], s["b"], s["y"], s["mean"], s["rstd"], stream=stream)
            return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
        m.layernorm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"], s["dx"], s["dw"], s["db"], s["workspace"],
                             dres=s["dres"], stream=stream)
        return {"dx": s["dx"], "dw": s["dw"], "db": s["db"]}
    if case["op"] == "logprobs":
        m.token_logprobs(s["logits"], s["targets"], s["logp"], s["entropy"], s["top_ids"], s["top_logp"], stream=stream)
        return {"logp": s["logp"], "entropy": s["entropy"], "top_ids": s["top_ids"], "top_logp": s["top_logp"]}
    m.distill_loss(s["logits"], s["top_ids"], s["top_logits"], s["loss"], s["lse"], temperature=case["temperature"],
                   stream=stream)
    m.distill_backward(s["logits"], s["top_ids"], s["top_logits"], s["lse"], s["dloss"], s["dlogits"],
                       temperature=case["temperature"], stream=stream)
    return {"loss": s["loss"], "dlogits": s["dlogits"]}


def _rows(cu, max_len):
    """Row of every place of the padded batch [B, max_len], and which places are tokens."""
    at = torch.arange(max_len, device=cu.device)
    start, length = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    valid = at[None] < length[:, None]
    return torch.where(valid, start[:, None] + at[None], 0), valid


def _heads(x, rows, valid, H):
    """[T, H dh] -> [B, H, max_len, dh] in 32 bits, zero where there is no token."""
    y = torch.where(valid[..., None], x[rows].float(), 0.0)
    return y.unflatten(-1, (H, -1)).transpose(1, 2)


def _attention_plain(s):
    case, H = s["case"], s["case"]["heads"]
    rows, valid = _rows(s["cu"], case["max_len"])
    q, k, v = (_heads(x, rows, valid, H) for x in s["qkv"].chunk(3, dim=1))
    scores = (q @ k.transpose(-1, -2)) / math.sqrt(case["head_dim"])
    scores = torch.where(valid[:, None, None, :], scores, -math.inf)
    top = torch.where(valid.any(1)[:, None, None, None], scores.amax(-1, keepdim=True), 0.0)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / total
    lse = (top + torch.log(total))[..., 0]
    return out.transpose(1, 2)[valid].flatten(1).to(s["qkv"].dtype), lse.transpose(1, 2)[valid].t().contiguous()


def _attention_backward_plain(s):
    case, H = s["case"], s["case"]["heads"]
    scale = 1.0 / math.sqrt(case["head_dim"])
    rows, valid = _rows(s["cu"], case["max_len"])
    q, k, v = (_heads(x, rows, valid, H) for x in s["qkv"].chunk(3, dim=1))
    out, dout = _heads(s["out"], rows, valid, H), _heads(s["dout"], rows, valid, H)
    lse = s["lse"].t()[rows].transpose(1, 2)
    both = valid[:, None, :, None] & valid[:, None, None, :]
    p = torch.where(both, torch.exp((q @ k.transpose(-1, -2)) * scale - lse[..., None]), 0.0)
    dv = p.transpose(-1, -2) @ dout
    dp = dout @ v.transpose(-1, -2)
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * scale
    grads = (ds @ k, ds.transpose(-1, -2) @ q, dv)
    return torch.cat([x.transpose(1, 2)[valid].flatten(1) for x in grads], dim=1).to(s["qkv"].dtype)


def _layernorm_plain(x, w, b, kind, eps=1e-5):
    x = x.float()
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((c * c).mean(1) + eps)
    return (c * rstd[:, None] * w + b).to(kind), mean, rstd


def _layernorm_backward_plain(s):
    x, dy = s["x"].float(), s["dy"].float()
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["w"]
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * xhat).sum(0), "db": dy.sum(0)}


def _logprobs_plain(s):
    x = s["logits"].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    lse = top + torch.log(e.sum(1, keepdim=True))
    logp = x - lse
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)  # ties go to the lowest index
    k = s["top_ids"].shape[1]
    return {"logp": logp.gather(1, s["targets"].long()[:, None])[:, 0], "entropy": entropy,
            "top_ids": ids[:, :k].to(torch.int32), "top_logp": best[:, :k] - lse}


def _distill_plain(s):
    tau, ids = s["case"]["temperature"], s["top_ids"].long()
    x = s["logits"].float() / tau
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    there = ids >= 0
    t = torch.where(there, s["top_logits"] / tau, -math.inf)
    t = t - t.amax(1, keepdim=True)
    logp = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    p = torch.exp(logp)
    at = torch.where(there, ids, 0)
    logq = x.gather(1, at) - lse
    loss = tau * tau * torch.where(there, p * (logp - logq), 0.0).sum(1)
    target = torch.zeros_like(x).scatter_add(1, at, p)
    dlogits = tau * s["dloss"][:, None] * (torch.exp(x - lse) - target)
    return {"loss": loss, "dlogits": dlogits.to(s["logits"].dtype)}


# ---- the same values in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "layernorm": _exact_layernorm, "logprobs": _exact_logprobs,
            "distill": _exact_distill}[case["op"]](case, s)


def _exact_attention(case, s):
    H, dh, cu = case["heads"], case["head_dim"], s["cu"].tolist()
    qkv = s["qkv"].view(-1, 3, H, dh)
    out = torch.empty(s["tokens"], H, dh, dtype=torch.float64, device="cuda")
    lse = torch.empty(H, s["tokens"], dtype=torch.float64, device="cuda")
    grad = torch.empty(s["tokens"], 3, H, dh, dtype=torch.float64, device="cuda")
    for a, b in zip(cu[:-1], cu[1:]):
        step = max(1, (1 << 27) // max(1, (b - a) ** 2))
        for h in range(0, H if b > a else 0, step):
            x = qkv[a:b, :, h:h + step].double().requires_grad_(case["way"] == "backward")
            scores = torch.einsum("ihd,jhd->hij", x[:, 0], x[:, 1]) / dh ** 0.5
            o = torch.einsum("hij,jhd->ihd", torch.softmax(scores, -1), x[:, 2])
            out[a:b, h:h + step], lse[h:h + step, a:b] = o.detach(), torch.logsumexp(scores.detach(), -1)
            if case["way"] == "backward":
                dout = s["dout"].view(-1, H, dh)[a:b, h:h + step].double()
                grad[a:b, :, h:h + step] = torch.autograd.grad(o, x, dout)[0]
    if case["way"] == "forward":
        return {"out": out.flatten(1), "lse": lse}
    return {"dqkv": grad.flatten(1)}


def _exact_layernorm(case, s):
    back = case["way"] == "backward"
    x, w, b = (s[n].double().requires_grad_(back) for n in ("x", "w", "b"))
    var, mean = torch.var_mean(x, dim=1, correction=0)
    y = (x - mean[:, None]) / torch.sqrt(var + 1e-5)[:, None] * w + b
    if not back:
        return {"y": y, "mean": mean, "rstd": (var + 1e-5).rsqrt()}
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return {"dx": dx if s["dres"] is None else dx + s["dres"].double(), "dw": dw, "db": db}


def _exact_logprobs(case, s):
    logp = torch.log_softmax(s["logits"].double(), dim=1)
    entropy = torch.special.entr(logp.exp()).sum(1)
    ids = torch.argsort(s["logits"].double(), dim=1, descending=True, stable=True)[:, :case["k"]]
    return {"logp": logp[torch.arange(case["rows"], device="cuda"), s["targets"].long()], "entropy": entropy,
            "top_ids": ids.to(torch.int32), "top_logp": torch.take_along_dim(logp, ids, 1)}


def _exact_distill(case, s):
    tau, V = case["temperature"], case["vocab"]
    x = s["logits"].double().requires_grad_()
    ids = s["top_ids"].long()
    teacher = torch.softmax(torch.where(ids >= 0, s["top_logits"].double(), -math.inf) / tau, dim=1)
    # The teacher's distribution over the vocabulary; one more column takes the absent alternatives.
    full = torch.zeros(case["rows"], V + 1, dtype=torch.float64, device="cuda")
    full = full.scatter_add(1, torch.where(ids >= 0, ids, V), teacher)[:, :V]
    logq = torch.log_softmax(x / tau, dim=1)
    loss = tau ** 2 * (torch.special.xlogy(full, full) - full * logq).sum(1)
    return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, x, s["dloss"].double())[0]}
