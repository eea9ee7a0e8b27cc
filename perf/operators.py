"""Operators of a training step that keep no [T, T] or [T, V] intermediate: their plain forms, and the cases they are timed at.

Causal attention over packed q, k, v rows, which saves the log of each row's softmax sum; its
backward pass, which computes the probabilities again from that; and the loss of a student
against a teacher's top logits and the hard targets, with its gradient.  `run` computes them
from elementary torch operations in fp32 where `own` is false, and through the library where
it is true.

Shapes: the Forge-98M and Forge-220M presets (12 heads of 64, contexts of 512 and 1024, a
vocabulary of 16257 or 16384), the 4-layer d-128 model of the known-answer tests (4 heads of
32, vocabulary 2256), and what is trained beside them: longer windows, heads of 128, shared
k and v heads, padded batches, larger vocabularies.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the known-answer model on a prompt's first ids: one launch, latency alone
        dict(name="attend_tiny", kind="attend", batch=1, rows=16, heads=4, kv_heads=4, head_dim=32, dtype="f32", ragged=False),
        # a micro-batch of Forge-98M at its context of 512
        dict(name="attend_98m", kind="attend", batch=4, rows=512, heads=12, kv_heads=12, head_dim=64, dtype="f32", ragged=False),
        # a padded batch of texts of their own lengths
        dict(name="attend_padded_bf16", kind="attend", batch=8, rows=777, heads=12, kv_heads=12, head_dim=64, dtype="bf16", ragged=True),
        # long windows of a model with heads of 128 that share k and v
        dict(name="attend_long_bf16", kind="attend", batch=2, rows=4096, heads=16, kv_heads=4, head_dim=128, dtype="bf16", ragged=False),
        # the known-answer model's training step
        dict(name="grad_tiny", kind="attend_grad", batch=2, rows=37, heads=4, kv_heads=4, head_dim=32, dtype="f32", ragged=False),
        # the micro-batch of Forge-98M again
        dict(name="grad_98m", kind="attend_grad", batch=4, rows=512, heads=12, kv_heads=12, head_dim=64, dtype="f32", ragged=False),
        # one long window in fp32, of a length that is no multiple of a tile
        dict(name="grad_long", kind="attend_grad", batch=1, rows=2500, heads=12, kv_heads=12, head_dim=64, dtype="f32", ragged=False),
        # full windows of 1024 in bf16
        dict(name="grad_98m_bf16", kind="attend_grad", batch=8, rows=1024, heads=12, kv_heads=12, head_dim=64, dtype="bf16", ragged=False),
        # heads of 128 that share k and v, padded
        dict(name="grad_shared_bf16", kind="attend_grad", batch=4, rows=1333, heads=16, kv_heads=4, head_dim=128, dtype="bf16", ragged=True),
        # the known-answer model scored against its teacher: the loss alone
        dict(name="distill_tiny", kind="distill", rows=16, vocab=2256, top=8, temperature=2.0, alpha=0.5, dtype="f32", grad=False),
        # the micro-batch of Forge-98M: loss and gradient over the released vocabulary (ragged rows)
        dict(name="distill_98m", kind="distill", rows=2048, vocab=16257, top=32, temperature=2.0, alpha=0.5, dtype="f32", grad=True),
        # a larger vocabulary in bf16 (odd, so that rows start anywhere), the teacher alone
        dict(name="distill_wide_bf16", kind="distill", rows=1500, vocab=50257, top=64, temperature=1.0, alpha=1.0, dtype="bf16", grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend_grad", "attend_grad", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "distill":
        vocab = rng.choice([2256, 4001, 16257, 16384, 32000, 50257])
        return dict(kind=kind, rows=_log(rng, 1, min(2048, 7.5e7 / vocab)), vocab=vocab, top=_log(rng, 1, 128),
                    temperature=rng.choice([1.0, 2.0, 4.0]), alpha=rng.choice([0.3, 0.5, 0.9, 1.0]), dtype=dtype,
                    grad=rng.random() < 0.7)
    hd = rng.choice([32, 40, 64, 64, 64, 80, 128])
    heads, kv = rng.choice([(4, 4), (8, 2), (12, 12), (12, 12), (12, 4), (16, 4)])
    most = 3.0e8 if dtype == "bf16" else 7.0e7  # scores of a pass: no more than the largest listed case's
    rows = _log(rng, 1, 4000 if dtype == "bf16" else 2400)
    batch = _log(rng, 1, max(1, min(16, 8192 // rows, most * 64 / max(64, hd) / (heads * rows * rows))))
    return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv, head_dim=hd, dtype=dtype,
                ragged=batch > 1 and rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------

def _attention_inputs(case, seed):
    """qkv rows, dO rows and each sequence's length (the first is full)."""
    B, T, H, Hk, hd = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    qkv = torch.randn(B * T, (H + 2 * Hk) * hd, generator=g, device="cuda").to(dt)
    dout = (torch.randn(B * T, H * hd, generator=g, device="cuda") * 1e-3).to(dt)
    lengths = np.full(B, T, np.int32)
    if case["ragged"]:
        lengths[1:] = np.random.default_rng(seed).integers(max(1, T // 8), T + 1, B - 1)
    return qkv, dout, lengths


def _distill_inputs(case, seed):
    """Student logits, host targets (some without a loss), and the teacher's top ids and logits.

    A teacher whose kept tokens are cut by probability leaves slots of a row empty: id -1."""
    T, V, K = case["rows"], case["vocab"], case["top"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(T, V, generator=g, device="cuda") * 2
    teacher = 0.7 * logits + torch.randn(T, V, generator=g, device="cuda") * 1.5
    top, ids = teacher.topk(K, dim=1)
    kept = torch.randint(1, 2 * K + 1, (T, 1), generator=g, device="cuda")
    empty = torch.arange(K, device="cuda") >= kept
    ids = ids.masked_fill(empty, -1).to(torch.int32)
    top = top.masked_fill(empty, 0.0)
    r = np.random.default_rng(seed)
    targets = np.where(r.random(T) < 0.7, ids[:, 0].cpu().numpy(), r.integers(0, V, T)).astype(np.int32)
    if T > 1:
        targets[1:][r.random(T - 1) < 0.05] = -1
    return logits.to(_DTYPES[case["dtype"]]), targets, ids.contiguous(), top.contiguous()


def prepare(case, seed):
    s = dict(case)
    if case["kind"] == "distill":
        s["logits"], s["targets"], s["ids"], s["top_logits"] = _distill_inputs(case, seed)
        s["dlogits"] = torch.empty_like(s["logits"]) if case["grad"] else None
    else:
        s["qkv"], s["dout"], s["lengths"] = _attention_inputs(case, seed)
        s["out"] = torch.empty_like(s["dout"])
        s["lse"] = torch.empty(case["batch"], case["heads"], case["rows"], device="cuda")
        s["dqkv"] = torch.empty_like(s["qkv"])
        if case["kind"] == "attend_grad":  # what the forward pass left
            s["out"], s["lse"] = _attend(s)
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------------------

_kept = {}


def _backend():
    """The process's device context, and the package, for the library's own calls."""
    if not _kept:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forge-lm_amd"))
        import forge_hip
        _kept["be"] = forge_hip.HipBackend(0)
    return _kept["be"]


def run(s):
    if s["kind"] == "distill":
        return _run_distill(s)
    return _run_attend(s) if s["kind"] == "attend" else _run_grad(s)


def _run_attend(s):
    if own:
        _backend().attention_forward(s["qkv"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(), s["batch"], s["rows"],
                                     s["heads"], s["head_dim"], n_kv_heads=s["kv_heads"],
                                     lengths=s["lengths"] if s["ragged"] else None, dtype=s["dtype"])
        return {"out": s["out"], "lse": s["lse"]}
    out, lse = _attend(s)
    return {"out": out, "lse": lse}


def _run_grad(s):
    if own:
        _backend().attention_backward(s["dout"].data_ptr(), s["qkv"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(),
                                      s["dqkv"].data_ptr(), s["batch"], s["rows"], s["heads"], s["head_dim"],
                                      n_kv_heads=s["kv_heads"], lengths=s["lengths"] if s["ragged"] else None,
                                      dtype=s["dtype"])
        return {"dqkv": s["dqkv"]}
    return {"dqkv": _attend_backward(s)}


def _run_distill(s):
    if own:
        loss = _backend().distill_loss(s["logits"].data_ptr(), s["targets"], s["ids"].data_ptr(), s["top_logits"].data_ptr(),
                                       s["dlogits"].data_ptr() if s["grad"] else None, s["rows"], s["vocab"], s["top"],
                                       ignore_index=-1, temperature=s["temperature"], alpha=s["alpha"], dtype=s["dtype"])
        return {"loss": loss, "dlogits": s["dlogits"]}
    loss, grad = _distill(s)
    return {"loss": float(loss), "dlogits": grad}


def _scores(s):
    """fp32 q [B, Hk, G, T, hd], k and v [B, Hk, 1, T, hd], scaled scores, and which of them count."""
    B, T, H, Hk, hd = (s[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim"))
    x = s["qkv"].float().view(B, T, H + 2 * Hk, hd).transpose(1, 2)
    q = x[:, :H].reshape(B, Hk, H // Hk, T, hd)
    k = x[:, H:H + Hk].unsqueeze(2).contiguous()
    v = x[:, H + Hk:].unsqueeze(2).contiguous()
    t = torch.arange(T, device="cuda")
    valid = t < torch.from_numpy(s["lengths"]).to("cuda").view(B, 1)
    seen = ((t <= t.view(T, 1)) & valid.view(B, 1, T) & valid.view(B, T, 1)).view(B, 1, 1, T, T)
    return q, k, v, torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd)), seen


def _attend(s):
    """Output rows [B * T, H * hd] and the log of each row's sum of exp(score) [B, H, T]."""
    B, T, H, hd = (s[k] for k in ("batch", "rows", "heads", "head_dim"))
    q, k, v, x, seen = _scores(s)
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(B, H, T, hd).transpose(1, 2).reshape(B * T, H * hd)
    return o.to(s["qkv"].dtype), (torch.log(total) + m).view(B, H, T)


def _attend_backward(s):
    """dQKV rows, with the probabilities computed again from the scores and the saved logs."""
    B, T, H, Hk, hd = (s[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim"))
    q, k, v, x, seen = _scores(s)
    heads = lambda a: a.float().view(B, T, H, hd).transpose(1, 2).reshape(B, Hk, H // Hk, T, hd)  # noqa: E731
    do, o = heads(s["dout"]), heads(s["out"])
    p = torch.where(seen, torch.exp(x - s["lse"].view(B, Hk, H // Hk, T, 1)), torch.zeros_like(x))
    del x
    valid = seen.any(-1, keepdim=True)
    do = torch.where(valid, do, torch.zeros_like(do))
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (ds - (do * o).sum(-1, keepdim=True)) * (1.0 / math.sqrt(hd))
    dq = torch.matmul(ds, k).view(B, H, T, hd)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).sum(2)
    return torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B * T, -1).to(s["qkv"].dtype)


def _distill(s):
    """Mean over the rows with a target of (1 - alpha) * cross-entropy + alpha * tau^2 * KL(teacher || student at
    tau), the teacher's distribution over its kept logits alone; and its gradient."""
    tau, alpha = s["temperature"], s["alpha"]
    z = s["logits"].float()
    target = torch.from_numpy(s["targets"]).to("cuda").long()
    on = target >= 0
    count = on.sum().clamp(min=1).double()
    target = target.clamp(min=0).view(-1, 1)
    used, ids = s["ids"] >= 0, s["ids"].clamp(min=0).long()

    def log_softmax(a):
        m = a.amax(-1, keepdim=True)
        return a - m - torch.log(torch.exp(a - m).sum(-1, keepdim=True))

    u = torch.where(used, s["top_logits"] / tau, torch.full_like(s["top_logits"], -1e30))
    q = torch.where(used, torch.exp(log_softmax(u)), torch.zeros_like(u))
    soft, hard = log_softmax(z / tau), log_softmax(z)
    kl = torch.where(used, q * (log_softmax(u) - soft.gather(1, ids)), torch.zeros_like(u)).sum(-1)
    row = (1 - alpha) * -hard.gather(1, target).view(-1) + alpha * tau * tau * kl
    loss = (torch.where(on, row, torch.zeros_like(row)).double().sum() / count).float()
    if not s["grad"]:
        return loss, None
    kept = used.any(-1, keepdim=True)
    g = torch.where(kept, torch.exp(soft), torch.zeros_like(soft)).scatter_add_(1, ids, -q) * (alpha * tau)
    hard = torch.exp(hard)
    hard.scatter_add_(1, target, -torch.ones_like(hard[:, :1]))
    g = torch.where(on.view(-1, 1), g + hard * (1 - alpha), torch.zeros_like(g)) / count.float()
    return loss, g.to(s["logits"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "distill":
        T, V, K = case["rows"], case["vocab"], case["top"]
        return {"bytes": float(e * T * V * (2 if case["grad"] else 1) + 8 * T * K + 4 * T), "flops": 12.0 * T * V}
    B, T, H, Hk, hd = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim"))
    # padded sequences by their mean length
    n = float(T)
    pairs = n * (n + 1) / 2
    if case["ragged"]:
        lo = max(1, T // 8)
        mean, square = (lo + T) / 2.0, (lo * lo + lo * T + T * T) / 3.0
        n, pairs = (T + (B - 1) * mean) / B, (pairs + (B - 1) * (square + mean) / 2) / B
    q, kv = B * H * hd, 2 * B * Hk * hd
    if case["kind"] == "attend":  # qkv read, O written (every row of it), the logs
        return {"bytes": e * (n * (q + kv) + T * q) + 4.0 * B * H * T, "flops": 4.0 * B * H * hd * pairs}
    # qkv, O and dO read, dQKV written, the logs read; the scores, dP and three gradients
    return {"bytes": e * (n * (3 * q + kv) + T * (q + kv)) + 4.0 * B * H * n, "flops": 10.0 * B * H * hd * pairs}


# ---- the same in 64 bits ---------------------------------------------------------------------------

def _one_head(q, k, v, n, T):
    """softmax(q k^T / sqrt(hd)) v of the first n rows of a sequence under the causal mask, zeros after."""
    w = (q[:n] @ k[:n].T) / math.sqrt(q.shape[1])
    w = w.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    lse = torch.logsumexp(w, 1)
    o = torch.softmax(w, 1) @ v[:n]
    return torch.cat([o, o.new_zeros(T - n, o.shape[1])]), torch.cat([lse, lse.new_full((T - n,), -math.inf)])


def exact(case, seed):
    if case["kind"] == "distill":
        return _exact_distill(case, seed)
    B, T, H, Hk, hd = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim"))
    qkv, dout, lengths = _attention_inputs(case, seed)
    x = qkv.double().view(B, T, H + 2 * Hk, hd)
    do = dout.double().view(B, T, H, hd)
    out = torch.zeros(B, T, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, H, T, dtype=torch.float64, device="cuda")
    grad = torch.zeros_like(x)
    for b in range(B):
        for h in range(H):
            at = (h, H + h // (H // Hk), H + Hk + h // (H // Hk))
            leaves = [x[b, :, i].clone().requires_grad_(True) for i in at]
            o, log_sum = _one_head(*leaves, int(lengths[b]), T)
            out[b, :, h], lse[b, h] = o.detach(), log_sum.detach()
            if case["kind"] == "attend_grad":
                for i, d in zip(at, torch.autograd.grad(o, leaves, do[b, :, h])):
                    grad[b, :, i] += d
    if case["kind"] == "attend":
        return {"out": out.view(B * T, -1), "lse": lse}
    return {"dqkv": grad.view(B * T, -1)}


def _exact_distill(case, seed):
    tau, alpha = case["temperature"], case["alpha"]
    logits, targets, ids, top = _distill_inputs(case, seed)
    z = logits.double().requires_grad_(True)
    rows = np.flatnonzero(targets >= 0)
    at = torch.from_numpy(rows).cuda()
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    if alpha < 1:
        ce = torch.nn.functional.cross_entropy(z[at], torch.from_numpy(targets[rows].astype(np.int64)).cuda(), reduction="sum")
        total = total + (1 - alpha) * ce
    teacher = torch.where(ids >= 0, top.double() / tau, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))[at]
    lq = torch.log_softmax(teacher, 1)
    lp = torch.log_softmax(z[at] / tau, 1).gather(1, ids[at].clamp(min=0).long())
    kl = torch.where(ids[at] >= 0, lq.exp() * (lq - lp), torch.zeros_like(lp)).sum()
    loss = (total + alpha * tau * tau * kl) / max(1, len(rows))
    if not case["grad"]:
        return {"loss": float(loss), "dlogits": None}
    return {"loss": float(loss), "dlogits": torch.autograd.grad(loss, z)[0]}
