"""Measured cases of the distillation operators: layer norm (forward, and forward with backward), a
teacher's top logits, and the distillation loss (alone, and with the gradient of the logits).

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the
end) while ``own`` is false, and through the framework's kernels while it is true.

Formulas (rows n, columns j):

  layer norm       xhat = (x - mean) rstd, rstd = 1 / sqrt(mean((x - mean)^2) + eps), y = xhat w + b
                   dx = rstd (g - mean(g) - xhat mean(g xhat)) with g = dy w,  dw = sum_n dy xhat,  db = sum_n dy
  top logits       the k largest logits of a row in descending order (ties: the lower column first), their
                   columns, and log sum_j exp(z_j / tau)
  distillation     p_i = exp(t_i / tau - L) over the teacher's listed columns, L the teacher's own log-sum-exp
                   (then m = 1 - sum p is the mass of all other columns) or that of its list (then m = 0);
                   q = softmax(z / tau);  q_rest = sum of q over the columns that are not listed
                   KL = sum_i p_i log(p_i / q_i) + m log(m / q_rest)
                   loss = scale (kd_weight tau^2 KL + ce_weight (-log softmax(z)_target))
                   rows whose target is negative count for nothing; list entries with a negative column are absent
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
LARGEST = 8192 * 65536 * 4  # bytes of the logits of the largest drawn case


def listed():
    ln = dict(op="layer_norm", bias=True)
    kd = dict(op="distill", masked=0.1)
    return [
        # one decoding step of eight sequences through a norm of the 1B shape: latency alone
        dict(ln, name="layer_norm_step", train=False, rows=8, d=2048, x="fp32", y="bf16"),
        # evaluation: the norm of one 8 x 2048 token micro-batch, fp32 residual stream to bf16 operand
        dict(ln, name="layer_norm_eval", train=False, rows=16384, d=2048, x="fp32", y="bf16"),
        # training: the same micro-batch forward and backward
        dict(ln, name="layer_norm_train", train=True, rows=16384, d=2048, x="fp32", y="bf16"),
        # training at the 32B width on a bf16 stream
        dict(ln, name="layer_norm_train_wide", train=True, rows=8192, d=6144, x="bf16", y="bf16"),
        # a ragged batch at an odd width, as small research models have
        dict(ln, name="layer_norm_train_odd", train=True, rows=3001, d=1037, x="fp32", y="fp32"),
        # the teacher's top logits of one token each of four sequences
        dict(op="top_logits", name="top_logits_step", rows=4, vocab=50257, ld=50304, k=32, tau=1.0, z="fp32"),
        # one loss chunk of a teacher's bf16 logits (50257 real columns of 50304)
        dict(op="top_logits", name="top_logits_chunk", rows=8192, vocab=50257, ld=50304, k=64, tau=2.0, z="bf16"),
        # a teacher with a large vocabulary, fp32 logits
        dict(op="top_logits", name="top_logits_large", rows=2048, vocab=131072, ld=131072, k=128, tau=1.0, z="fp32"),
        # a test-sized student: 64 tokens of a small vocabulary
        dict(kd, name="distill_train_small", train=True, rows=64, vocab=500, ld=512, k=8, tau=1.0, ce=0.5, rest=True,
             z="fp32"),
        # evaluation of a student against stored teacher logits
        dict(kd, name="distill_eval", train=False, rows=4096, vocab=50257, ld=50304, k=64, tau=1.0, ce=0.0, rest=True,
             z="bf16"),
        # training: one loss chunk, softened teacher renormalised over its list, mixed with cross-entropy
        dict(kd, name="distill_train_chunk", train=True, rows=8192, vocab=50257, ld=50304, k=64, tau=2.0, ce=0.25,
             rest=False, z="bf16"),
        # training with fp32 logits and a large vocabulary, the mass beyond the teacher's list kept
        dict(kd, name="distill_train_large", train=True, rows=4096, vocab=131072, ld=131072, k=128, tau=1.0, ce=0.0,
             rest=True, z="fp32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "top_logits", "distill"])
    if op == "layer_norm":
        d = _log_uniform(rng, 64, 8192)
        if rng.random() < 0.6:
            d = max(64, d // 64 * 64)
        rows = min(_log_uniform(rng, 1, 32768), 16384 * 6144 // d)
        x = rng.choice(["fp32", "bf16", "fp16"])
        return dict(op=op, train=rng.random() < 0.6, rows=rows, d=d, x=x, y=rng.choice([x, "bf16"]) if x == "fp32" else x,
                    bias=rng.random() < 0.8)
    z = rng.choice(["fp32", "bf16", "fp16"])
    vocab = _log_uniform(rng, 256, 131072)
    ld = vocab if rng.random() < 0.5 else -(-vocab // 64) * 64
    rows = min(_log_uniform(rng, 1, 16384), LARGEST // (ld * BYTES[z]))
    k = _log_uniform(rng, 1, 128)
    tau = rng.choice([1.0, 1.0, 1.5, 2.0, 4.0])
    if op == "top_logits":
        return dict(op=op, rows=min(rows, 268435456 // ld), vocab=vocab, ld=ld, k=k, tau=tau, z=z)
    return dict(op=op, train=rng.random() < 0.7, rows=rows, vocab=vocab, ld=ld, k=k, tau=tau,
                ce=rng.choice([0.0, 0.1, 0.5]), rest=rng.random() < 0.5, z=z, masked=rng.choice([0.0, 0.1, 0.3]))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)
    rand = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    s = {"case": case}
    n = case["rows"]
    if case["op"] == "layer_norm":
        d = case["d"]
        # a residual stream: token scales that differ, a few large features, a mean that is not zero
        x = rand(n, d) * (0.5 + 2 * torch.rand(n, 1, device=dev, generator=g)) + 0.3 * rand(1, d)
        x[:, :: max(1, d // 7)] *= 6.0
        s["x"] = x.to(DTYPES[case["x"]]).requires_grad_(case["train"])
        s["w"] = (1 + 0.2 * rand(d)).requires_grad_(case["train"])
        s["b"] = (0.1 * rand(d)).requires_grad_(case["train"]) if case["bias"] else None
        if case["train"]:
            s["dy"] = (rand(n, d) * 0.02).to(DTYPES[case["y"]])
        return s
    v, ld, k = case["vocab"], case["ld"], min(case["k"], case["vocab"])
    dt = DTYPES[case["z"]]
    z = torch.empty(n, ld, device=dev, dtype=dt)
    if case["op"] == "top_logits":
        offset = 1.5 * rand(1, ld)  # frequent and rare tokens
        for r in range(0, n, 4096):  # in pieces: the fp32 draw of a piece stays small
            z[r:r + 4096] = (2.2 * rand(min(4096, n - r), ld) + offset).to(dt)
        s["z"], s["k"] = z[:, :v], k
        return s
    for r in range(0, n, 4096):
        z[r:r + 4096] = (1.6 * rand(min(4096, n - r), ld)).to(dt)
    # the teacher's list: distinct columns anywhere in the vocabulary, logits that fall off, and a
    # student that has learned part of it
    start = torch.randint(0, v, (n, 1), device=dev, generator=g)
    step = next(q for q in (7919, 6007, 4001, 1009, 101, 1) if math.gcd(q, v) == 1)
    ids = (start + torch.arange(k, device=dev) * step) % v
    gaps = torch.empty(n, k, device=dev).exponential_(3.0, generator=g)
    t = (11.0 - gaps.cumsum(1)).to(dt)
    z.scatter_(1, ids, (0.7 * t.float() + 0.8 * rand(n, k)).to(dt))
    absent = torch.rand(n, k, device=dev, generator=g) < 0.05  # entries a teacher left out
    absent |= torch.rand(n, 1, device=dev, generator=g) < 0.02  # rows without any entry
    s["ids"] = torch.where(absent, torch.full_like(ids, -1), ids).to(torch.int32)
    s["t"] = t
    soft = t.float() / case["tau"]
    beyond = 0.02 + 0.3 * torch.rand(n, device=dev, generator=g)  # the teacher's mass outside its list
    s["lse"] = torch.logsumexp(soft, 1) + torch.log1p(beyond) if case["rest"] else None
    target = torch.randint(0, v, (n,), device=dev, generator=g)
    hit = torch.rand(n, device=dev, generator=g) < 0.5
    target = torch.where(hit, ids[:, 0], target)
    ignored = torch.rand(n, device=dev, generator=g) < case["masked"]
    s["targets"] = torch.where(ignored, torch.full_like(target, -100), target)
    loss_scale = 8192.0 if case["z"] == "fp16" else 1.0  # as fp16 training has it: its gradients would vanish
    s["scale"] = loss_scale / (~ignored).sum().clamp_min(1).float()
    s["z"] = z[:, :v].requires_grad_(case["train"])
    return s


# ------------------------------------------------------------------------------------ plain forms
def _plain_layer_norm(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["w"].detach()
    xc = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
    xhat = xc * rstd
    y = xhat * w
    if s["b"] is not None:
        y = y + s["b"].detach()
    out = [y.to(DTYPES[case["y"]])]
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        out += [dx.to(s["x"].dtype), (dy * xhat).sum(0)]
        if s["b"] is not None:
            out.append(dy.sum(0))
    return out


def _plain_top_logits(s):
    z, k, tau = s["z"], s["k"], s["case"]["tau"]
    zf = z.float()
    # one whole number per element, larger for a larger value and, among equal values, for a lower column
    bits = (zf + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    column = torch.arange(z.shape[1], device=z.device)
    key = (order << 32) | (0x7FFFFFFF - column)
    ids = 0x7FFFFFFF - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    soft = zf / tau
    top = soft.amax(1, keepdim=True)
    lse = torch.log(torch.exp(soft - top).sum(1)) + top.squeeze(1)
    return [z.gather(1, ids), ids.to(torch.int32), lse]


def _plain_distill(s):
    case = s["case"]
    tau, ce = case["tau"], case["ce"]
    z = s["z"].detach().float()
    n, v = z.shape
    ids, t = s["ids"].long(), s["t"].float() / tau
    present = ids >= 0
    some = present.any(1)
    at = torch.where(present, ids, torch.zeros_like(ids))
    live = (s["targets"] >= 0).float() * s["scale"]
    if s["lse"] is not None:
        logp = t - s["lse"].unsqueeze(1)
        p = torch.where(present, torch.exp(logp), torch.zeros_like(t))
        m = torch.where(some, (1 - p.sum(1)).clamp_min(0), torch.zeros_like(live))
    else:
        masked = torch.where(present, t, torch.full_like(t, -math.inf))
        top = torch.where(some, masked.amax(1), torch.zeros_like(live)).unsqueeze(1)
        e = torch.exp(masked - top)
        total = torch.where(some, e.sum(1), torch.ones_like(live)).unsqueeze(1)
        logp, p = t - top - torch.log(total), e / total
        m = torch.zeros_like(live)
    soft = z / tau
    top = soft.amax(1, keepdim=True)
    e = torch.exp(soft - top)
    total = e.sum(1, keepdim=True)
    logq = soft.gather(1, at) - top - torch.log(total)
    kl = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
    listed = torch.zeros(n, v + 1, device=z.device, dtype=torch.bool)
    listed.scatter_(1, torch.where(present, ids, torch.full_like(ids, v)), True)
    listed = listed[:, :v]
    if s["lse"] is not None:
        q_rest = torch.where(listed, torch.zeros_like(e), e).sum(1) / total.squeeze(1)
        has = m > 0
        kl = kl + torch.where(has, m * torch.log(torch.where(has, m / q_rest, torch.ones_like(m))), torch.zeros_like(m))
    loss = tau * tau * kl
    target = s["targets"].clamp_min(0).unsqueeze(1)
    if ce:
        top1 = z.amax(1, keepdim=True)
        total1 = torch.exp(z - top1).sum(1, keepdim=True)
        loss = loss + ce * (top1 + torch.log(total1) - z.gather(1, target)).squeeze(1)
    loss = torch.where(live > 0, loss * live, torch.zeros_like(loss))
    if not case["train"]:
        return [loss]
    q = e / total
    mass = (p.sum(1) + m).unsqueeze(1)
    grad = q * mass
    if s["lse"] is not None:
        grad = grad - torch.where(listed, torch.zeros_like(q), q * (m / q_rest).unsqueeze(1))
    grad.scatter_add_(1, at, -p)
    grad = grad * tau
    if ce:
        grad += ce * torch.exp(z - top1) / total1
        grad.scatter_add_(1, target, torch.full_like(target, -ce, dtype=grad.dtype))
    grad = torch.where((live > 0).unsqueeze(1), grad * live.unsqueeze(1), torch.zeros_like(grad))
    return [loss.sum(), grad.to(s["z"].dtype)]


PLAIN = {"layer_norm": _plain_layer_norm, "top_logits": _plain_top_logits, "distill": _plain_distill}


# ------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    case = s["case"]
    if case["op"] == "layer_norm":
        from tensor_train_ing_b200.ops.layer_norm import layer_norm
        y = layer_norm(s["x"], s["w"], s["b"], eps=1e-5, out_dtype=DTYPES[case["y"]])
        if not case["train"]:
            return [y]
        wrt = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, wrt, s["dy"])]
    if case["op"] == "top_logits":
        from tensor_train_ing_b200.ops.distill import top_logits
        return list(top_logits(s["z"], s["k"], temperature=case["tau"]))
    from tensor_train_ing_b200.ops.distill import distillation_loss
    args = dict(teacher_lse=s["lse"], targets=s["targets"], temperature=case["tau"], ce_weight=case["ce"],
                scale=s["scale"])
    if not case["train"]:
        return [distillation_loss(s["z"], s["ids"], s["t"], reduction="none", **args)]
    loss = distillation_loss(s["z"], s["ids"], s["t"], **args)
    return [loss.detach(), *torch.autograd.grad(loss, s["z"])]


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


def work(case):
    n = case["rows"]
    if case["op"] == "layer_norm":
        d, bx, by = case["d"], BYTES[case["x"]], BYTES[case["y"]]
        vectors = 2 if case["bias"] else 1
        if not case["train"]:
            return {"bytes": n * d * (bx + by) + 4 * d * vectors, "flops": 7 * n * d}
        # forward: x in, y out; backward: dy in, dx out, the two parameter gradients
        return {"bytes": n * d * (bx + by + by + bx) + 8 * d * vectors, "flops": 18 * n * d}
    v, k, bz = case["vocab"], min(case["k"], case["vocab"]), BYTES[case["z"]]
    if case["op"] == "top_logits":
        return {"bytes": n * (v * bz + k * (bz + 4) + 4), "flops": 4 * n * v}
    teacher = n * (k * (bz + 4) + 8 + (4 if case["rest"] else 0))
    sums = 2 if case["ce"] and case["tau"] != 1.0 else 1
    grads = 2 if case["train"] else 1
    return {"bytes": n * v * bz * grads + teacher + 4 * n, "flops": 4 * n * v * sums * grads}


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _exact_layer_norm, "top_logits": _exact_top_logits, "distill": _exact_distill}[case["op"]](s)


def _exact_layer_norm(s):
    x = s["x"].detach().double().requires_grad_(True)
    w = s["w"].detach().double().requires_grad_(True)
    b = s["b"].detach().double().requires_grad_(True) if s["b"] is not None else None
    var, mean = torch.var_mean(x, dim=1, keepdim=True, unbiased=False)
    y = (x - mean) / torch.sqrt(var + 1e-5) * w
    if b is not None:
        y = y + b
    if not s["case"]["train"]:
        return [y.detach()]
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s["dy"].double())
    return [y.detach(), *grads]


def _exact_top_logits(s):
    lse = torch.cat([torch.logsumexp(piece.double() / s["case"]["tau"], 1) for piece in s["z"].split(1024)])
    return [None, None, lse]


def _exact_distill(s):
    """Piece by piece over rows: log-probabilities, the loss, and its gradient by autograd."""
    case = s["case"]
    tau = case["tau"]
    losses, grads = [], []
    for lo in range(0, case["rows"], 512):
        part = slice(lo, lo + 512)
        z = s["z"][part].detach().double().requires_grad_(True)
        ids = s["ids"][part].long()
        t = s["t"][part].double() / tau
        keep = ids >= 0
        logq = torch.log_softmax(z / tau, 1)
        blank = t.masked_fill(~keep, -math.inf)
        norm = s["lse"][part].double() if s["lse"] is not None else torch.logsumexp(blank, 1)
        norm = torch.where(keep.any(1), norm, torch.zeros_like(norm)).unsqueeze(1)
        logp = blank - norm
        p = logp.exp()
        kl = (p * (logp.masked_fill(~keep, 0.0) - logq.gather(1, ids.clamp_min(0)))).sum(1)
        if s["lse"] is not None:
            m = (1 - p.sum(1)).clamp_min(0) * keep.any(1)
            others = torch.ones_like(z, dtype=torch.bool)
            rows, cols = keep.nonzero(as_tuple=True)
            others[rows, ids[rows, cols]] = False
            rest = torch.logsumexp(logq.masked_fill(~others, -math.inf), 1)
            kl = kl + torch.where(m > 0, m * (torch.log(m.clamp_min(1e-300)) - rest), torch.zeros_like(m))
        loss = tau ** 2 * kl
        target = s["targets"][part]
        if case["ce"]:
            loss = loss - case["ce"] * torch.log_softmax(z, 1).gather(1, target.clamp_min(0).unsqueeze(1)).squeeze(1)
        loss = torch.where(target >= 0, loss, torch.zeros_like(loss)) * s["scale"].double()
        losses.append(loss.detach())
        if case["train"]:
            grads.append(torch.autograd.grad(loss.sum(), z)[0])
    loss = torch.cat(losses)
    return [loss.sum(), torch.cat(grads)] if case["train"] else [loss]
