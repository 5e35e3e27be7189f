"""What the operators of a student's training step cost: embedding lookup and its gradient, the gated feed-forward block, distillation.

A student is trained on a teacher's top logits: token or node ids are looked up in a table (`embedding`, `embedding_grad`), rows pass
through a gated feed-forward block (`gated_ffn`, `gated_ffn_grad`), and the logits are held to the teacher's (`distill`, `distill_grad`,
`distill_loss_grad`).  `run` computes one call of such an operator in plain torch operations, or, where `own` is true, through
graphslim_amd.ops.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one step of serving: the ids of a few sequences
        {"name": "lookup_step_bf16", "op": "lookup", "type": "bf16", "rows": 32000, "width": 1024, "tokens": 8},
        # a training batch's ids, padded at the ends of its sequences
        {"name": "lookup_batch_f32", "op": "lookup", "type": "f32", "rows": 50001, "width": 602, "tokens": 16383},
        # the table's gradient for a small vocabulary of odd size
        {"name": "lookup_grad_f32", "op": "lookup_grad", "type": "f32", "rows": 10007, "width": 500, "tokens": 5001},
        # the table's gradient for a large vocabulary and batch
        {"name": "lookup_grad_bf16", "op": "lookup_grad", "type": "bf16", "rows": 128000, "width": 2048, "tokens": 32768},
        # one token of serving: the weights are all there is to read
        {"name": "gated_step_bf16", "op": "gated", "type": "bf16", "rows": 1, "width": 2048, "inner": 8192, "act": "silu"},
        # a prompt of ragged length over features whose rows are not 16-byte aligned
        {"name": "gated_prompt_f16", "op": "gated", "type": "f16", "rows": 999, "width": 1433, "inner": 4096, "act": "gelu"},
        # forward and backward of a training batch
        {"name": "gated_train_bf16", "op": "gated_train", "type": "bf16", "rows": 8192, "width": 2048, "inner": 8192, "act": "silu"},
        # forward and backward in 32 bits at a citation graph's sizes
        {"name": "gated_train_f32", "op": "gated_train", "type": "f32", "rows": 2708, "width": 500, "inner": 1024, "act": "silu"},
        # a condensed graph's rows and classes
        {"name": "distill_graph_f32", "op": "distill_train", "type": "f32", "rows": 454, "classes": 40, "top": 5, "tau": 2.0},
        # loss and gradient of a training batch in one call
        {"name": "distill_train_bf16", "op": "distill_train", "type": "bf16", "rows": 8192, "classes": 32000, "top": 64, "tau": 1.0},
        # the loss alone, as a validation pass has it, over a large odd vocabulary
        {"name": "distill_loss_f16", "op": "distill", "type": "f16", "rows": 2047, "classes": 100003, "top": 20, "tau": 1.5},
        # the gradient alone, where the loss was computed before (gradient accumulation, re-weighted rows)
        {"name": "distill_grad_f32", "op": "distill_grad", "type": "f32", "rows": 1024, "classes": 50001, "top": 128, "tau": 2.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "gated", "gated_train", "distill", "distill_grad", "distill_train"])
    typ = rng.choice(["f32", "f16", "bf16"])
    if op in ("lookup", "lookup_grad"):
        return {"op": op, "type": typ, "rows": _log_int(rng, 100, 128000), "width": _log_int(rng, 16, 2048), "tokens": _log_int(rng, 1, 32768)}
    if op in ("gated", "gated_train"):
        # 32-bit products cost many times what 16-bit ones do: a shorter batch keeps them below the largest listed case
        rows = _log_int(rng, 1, 8192 if typ != "f32" else 1024)
        width, inner = _log_int(rng, 32, 2048), _log_int(rng, 64, 8192)
        if rng.random() < 0.5:  # half of the layers in use have widths of whole cache lines
            width, inner = max(64, width // 64 * 64), max(64, inner // 64 * 64)
        # relu's gradient jumps at 0, where rounding alone decides the side a pre-activation falls on: forward only
        act = rng.choice(["silu", "gelu", "sigmoid"] + ["relu"] * (op == "gated"))
        return {"op": op, "type": typ, "rows": rows, "width": width, "inner": inner, "act": act}
    classes = _log_int(rng, 7, 131072)
    rows = _log_int(rng, 1, max(1, min(8192, 8192 * 16000 // classes)))
    return {"op": op, "type": typ, "rows": rows, "classes": classes, "top": min(classes, _log_int(rng, 1, 128)),
            "tau": rng.choice([1.0, 1.5, 2.0, 4.0])}


def _ids(g, n, rows):
    """Ids as text has them, rank r with a share of 1 / r, a tenth of them padding (-1)."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    ids = (ids * 7919 + 13) % rows if rows % 7919 else ids  # frequent ids anywhere in the table
    return torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, torch.full_like(ids, -1), ids).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    t = _TYPES[case["type"]]
    op, n = case["op"], case["rows"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)

    s = dict(case)
    if op in ("lookup", "lookup_grad"):
        s["ids"] = _ids(g, case["tokens"], n)
        s["scale"] = math.sqrt(case["width"])
        if op == "lookup":
            s["table"] = normal(n, case["width"], std=0.02)
        else:
            s["d_out"] = normal(case["tokens"], case["width"], std=0.01)
    elif op in ("gated", "gated_train"):
        d, f = case["width"], case["inner"]
        s["x"] = normal(n, d)
        s["w_gate"], s["w_up"] = normal(f, d, std=d ** -0.5), normal(f, d, std=d ** -0.5)
        if op == "gated_train":
            s["d_h"] = normal(n, f, std=0.1)
    else:
        v, k = case["classes"], case["top"]
        first = torch.rand(n, 1, generator=g, device="cuda")
        step = 1 + (torch.rand(n, 1, generator=g, device="cuda") * max(0, v // k - 1)).long()
        at = ((first * v).long() + step * torch.arange(k, device="cuda")) % v  # k different classes a row
        val = torch.sort(torch.randn(n, k, generator=g, device="cuda") * 3 + 4, dim=1, descending=True).values
        have = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.1, 0.0, torch.rand(n, 1, generator=g, device="cuda") * 0.5 + 0.75)
        gone = torch.arange(k, device="cuda") >= (have * k).ceil()  # padded rows have no teacher, some rows a shorter list
        z = torch.randn(n, v, generator=g, device="cuda") * 2
        z.scatter_add_(1, at, 0.5 * val + torch.randn(n, k, generator=g, device="cuda"))
        s["logits"], s["top_values"] = z.to(t), val.to(t)
        s["top_ids"] = torch.where(gone, -1, at).to(torch.int32)
        # mean over the batch; gradients in fp16 are kept in range by a loss scale, as fp16 training has it
        s["d_loss"] = torch.full((n,), (32768.0 if case["type"] == "f16" else 1.0) / n, device="cuda")
        if op == "distill_grad":  # what the forward call left for the backward one
            s["lse"] = torch.logsumexp(s["logits"].double() / case["tau"], 1).float()
    return s


def _act(name, g):
    """The activation and its derivative."""
    if name == "relu":
        on = (g > 0).to(g.dtype)
        return torch.where(g > 0, g, 0.0), on
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-g))
    if name == "silu":
        return g * sig, sig * (1 + g * (1 - sig))
    return sig, sig * (1 - sig)


def _lookup(s):
    ids, rows = s["ids"], s["rows"]
    ok = (ids >= 0) & (ids < rows)
    got = s["table"][ids.clamp(0, rows - 1).long()].float() * s["scale"]
    return torch.where(ok[:, None], got, 0.0).to(s["table"].dtype)


def _lookup_grad(s):
    ids, rows, d = s["ids"], s["rows"], s["d_out"]
    ok = (ids >= 0) & (ids < rows)
    sums = torch.zeros(rows + 1, d.shape[1], device=d.device)
    sums.index_add_(0, torch.where(ok, ids, rows), d.float())
    return (sums[:rows] * s["scale"]).to(d.dtype)


def _gated(s, train):
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(s["act"], g)
    t = s["x"].dtype
    h = (a * u).to(t)
    if not train:
        return h
    d_h = s["d_h"].float()
    dg, du = d_h * u * da, d_h * a
    return {"h": h, "d_x": (dg @ wg + du @ wu).to(t), "d_w_gate": (dg.T @ x).to(t), "d_w_up": (du.T @ x).to(t)}


def _teacher(s):
    """(has a place, its class, log p, p) for each of the teacher's entries; softmax over a row's entries."""
    at, tau = s["top_ids"], s["tau"]
    ok = (at >= 0) & (at < s["classes"])
    v = torch.where(ok, s["top_values"].float() / tau, -math.inf)
    top = v.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(v - top)
    total = e.sum(1, keepdim=True)
    logp = v - top - torch.log(total)
    return ok, at.clamp(0, s["classes"] - 1).long(), logp, torch.where(total > 0, e / total, 0.0)


def _distill(s, loss, grad):
    tau = s["tau"]
    z = s["logits"].float() / tau
    ok, at, logp, p = _teacher(s)
    if loss:
        top = z.amax(1, keepdim=True)
        lse = torch.log(torch.exp(z - top).sum(1)) + top[:, 0]
        logq = z.gather(1, at) - lse[:, None]
        rows = tau * tau * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    else:
        lse = s["lse"]
    if not grad:
        return {"loss": rows, "lse": lse}
    w = s["d_loss"] * tau * ok.any(1)
    d = torch.exp(z - lse[:, None]) * w[:, None]
    d.scatter_add_(1, at, -p * w[:, None])
    d = d.to(s["logits"].dtype)
    return {"loss": rows, "d_logits": d} if loss else d


def _run_own(s):
    from graphslim_amd import ops

    op = s["op"]
    if op == "lookup":
        return ops.embedding(s["table"], s["ids"], s["scale"])
    if op == "lookup_grad":
        return ops.embedding_grad(s["d_out"], s["ids"], s["rows"], s["scale"])
    if op == "gated":
        return ops.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["act"])
    if op == "gated_train":
        h, saved = ops.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["act"], save=True)
        d_x, d_wg, d_wu = ops.gated_ffn_grad(s["d_h"], s["x"], s["w_gate"], s["w_up"], saved, s["act"])
        return {"h": h, "d_x": d_x, "d_w_gate": d_wg, "d_w_up": d_wu}
    if op == "distill":
        loss, lse = ops.distill(s["logits"], s["top_values"], s["top_ids"], s["tau"])
        return {"loss": loss, "lse": lse}
    if op == "distill_grad":
        return ops.distill_grad(s["logits"], s["top_values"], s["top_ids"], s["lse"], s["d_loss"], s["tau"])
    loss, d_logits = ops.distill_loss_grad(s["logits"], s["top_values"], s["top_ids"], s["d_loss"], s["tau"])
    return {"loss": loss, "d_logits": d_logits}


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "lookup":
        return _lookup(state)
    if op == "lookup_grad":
        return _lookup_grad(state)
    if op in ("gated", "gated_train"):
        return _gated(state, op == "gated_train")
    return _distill(state, op != "distill_grad", op != "distill")


def work(case):
    b, n, op = _BYTES[case["type"]], case["rows"], case["op"]
    if op in ("lookup", "lookup_grad"):
        t, f = case["tokens"], case["width"]
        if op == "lookup_grad":
            return {"bytes": t * f * b + 4 * t + n * f * b, "flops": t * f}
        share = np.diff(np.log(np.arange(1.0, n + 2))) / math.log(n + 1.0) * 0.9
        distinct = float(np.sum(-np.expm1(t * np.log1p(-share))))  # rows that are expected to be looked up at all
        return {"bytes": distinct * f * b + 4 * t + t * f * b, "flops": t * f}
    if op in ("gated", "gated_train"):
        d, f = case["width"], case["inner"]
        if op == "gated":
            return {"bytes": (n * d + 2 * f * d + n * f) * b, "flops": 4 * n * d * f}
        return {"bytes": (n * d + 2 * f * d + n * f + n * f + n * d + 2 * f * d) * b, "flops": 12 * n * d * f}
    v, k = case["classes"], case["top"]
    read = n * v * b + n * k * (b + 4)
    more = {"distill": 8 * n, "distill_grad": n * v * b + 8 * n, "distill_train": n * v * b + 8 * n}[op]
    return {"bytes": read + more, "flops": 4 * n * v}


def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], case["rows"]
    if op in ("lookup", "lookup_grad"):
        ids, f = s["ids"].long(), case["width"]
        inside = torch.nonzero((ids >= 0) & (ids < n))[:, 0]
        if op == "lookup":
            out = torch.zeros(case["tokens"], f, dtype=torch.float64, device="cuda")
            out[inside] = s["table"].double()[ids[inside]] * s["scale"]
            return out
        out = torch.zeros(n, f, dtype=torch.float64, device="cuda")
        out.index_put_((ids[inside],), s["d_out"].double()[inside] * s["scale"], accumulate=True)
        return out
    if op in ("gated", "gated_train"):
        x, wg, wu = (s[k].double() for k in ("x", "w_gate", "w_up"))
        g, u = torch.mm(x, wg.t().contiguous()), torch.mm(x, wu.t().contiguous())
        name = case["act"]
        if name == "relu":
            a, slope = torch.clamp(g, min=0), torch.heaviside(g, torch.zeros_like(g))
        elif name == "gelu":
            lower = 0.5 * torch.erfc(-g / math.sqrt(2.0))
            a, slope = g * lower, lower + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        else:
            lower = torch.sigmoid(g)
            a, slope = (g * lower, lower + g * lower * torch.sigmoid(-g)) if name == "silu" else (lower, lower * torch.sigmoid(-g))
        if op == "gated":
            return a * u
        d_h = s["d_h"].double()
        d_g, d_u = d_h * u * slope, d_h * a
        return {"h": a * u, "d_x": torch.mm(d_g, wg) + torch.mm(d_u, wu), "d_w_gate": torch.mm(d_g.t().contiguous(), x),
                "d_w_up": torch.mm(d_u.t().contiguous(), x)}
    tau, v = case["tau"], case["classes"]
    ids = s["top_ids"].long()
    there = (ids >= 0) & (ids < v)
    any_there = there.any(1)
    t = s["top_values"].double() / tau
    t = torch.where(there, t, torch.full_like(t, -math.inf))
    t = torch.where(any_there[:, None], t, torch.zeros_like(t))  # rows without a teacher are left out below
    logp = torch.log_softmax(t, 1)
    p = torch.where(there, torch.exp(logp), torch.zeros_like(t))
    z = s["logits"].double() / tau
    lse = torch.logsumexp(z, 1)
    q_at = torch.take_along_dim(z, torch.where(there, ids, torch.zeros_like(ids)), 1) - lse[:, None]
    loss = tau * tau * torch.where(p > 0, p * (logp - q_at), torch.zeros_like(p)).sum(1)
    if op == "distill":
        return {"loss": loss, "lse": lse}
    z -= lse[:, None]
    d = z.exp_()
    d *= (s["d_loss"].double() * tau * any_there)[:, None]
    row = torch.arange(n, device="cuda")[:, None].expand_as(ids)
    d.index_put_((row[there], ids[there]), -(p * (s["d_loss"].double() * tau)[:, None])[there], accumulate=True)
    return d if op == "distill_grad" else {"loss": loss, "d_logits": d}
