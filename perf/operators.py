"""Performance cases of the operators at the two ends of a student's training step: the embedding with its gradient, a
teacher's top logits, and the distillation loss with its gradient.

A case is a dict of plain values. Its ``kind`` selects the operator:

  * "emb":     embedding(idx, weight, scale, padding_idx): the lookup, and with ``train`` the weight's gradient. ``ids``
    says how the tokens are spread: "zipf" (text), "uniform" (the training command's synthetic stream), "one" (a batch of
    padding or of one repeated token: every gradient row meets in one row of the weight).
  * "top":     top_logits(logits, k, temperature): a frozen teacher's evaluation.
  * "distill": distill_loss(logits, values, indices, rest, targets, temperature, weight): the loss, and with ``train`` the
    logits' gradient. ``rest``: the teacher's remaining mass is a class of its own; ``hard``: targets are given (rows whose
    target is -100 are left out), with 1 - weight of the loss their cross entropy.

``shift`` takes logits[:, :-1] of one position more per sequence, as a program does whose targets are the inputs.

The sizes are those of this repository's model (d_model 768, vocabulary 50304, B = 8 and 32, T = 1024 and 256), of its tests
(vocabularies 512 and 1003, small ragged batches) and generic ones (vocabulary 32000). ``draw`` spreads over the same ranges.
"""

import functools
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_MOST = 8192 * 50304  # logits of the largest case
_MOST_EMB = 131072 * 768  # gradient values of the largest embedding case


def listed():
    return [
        # The smallest call: one short prompt's embedding, where launch latency is the time.
        dict(name="emb_fwd_256x768", kind="emb", train=False, B=1, T=256, V=50304, N=768, dtype="fp32", ids="zipf", scale=1.0, pad=False),
        # The model's embedding in one training step (B = 8, T = 1024) on text, forward and gradient.
        dict(name="emb_train_8192x768", kind="emb", train=True, B=8, T=1024, V=50304, N=768, dtype="fp32", ids="zipf", scale=1.0, pad=False),
        # A large batch in 16 bits with scaled embeddings: gradients of 131072 tokens.
        dict(name="emb_train_131072x768_bf16", kind="emb", train=True, B=128, T=1024, V=50304, N=768, dtype="bf16", ids="zipf", scale=27.712812921102035, pad=True),
        # An odd width, a small vocabulary and a batch of one token: all gradients meet in one row.
        dict(name="emb_train_one_token_fp16", kind="emb", train=True, B=5, T=777, V=1003, N=203, dtype="fp16", ids="one", scale=1.0, pad=False),
        # A teacher's next-token logits for one sequence.
        dict(name="top_1x50304_k64", kind="top", B=1, T=1, V=50304, k=64, dtype="bf16", tau=1.0, shift=False),
        # A teacher's evaluation of the model's training batch.
        dict(name="top_8192x50304_k64", kind="top", B=8, T=1024, V=50304, k=64, dtype="bf16", tau=2.0, shift=False),
        # Many logits kept, fp32, shifted rows.
        dict(name="top_2044x32000_k256_fp32", kind="top", B=4, T=511, V=32000, k=256, dtype="fp32", tau=1.0, shift=True),
        # The loss of one training step at the model's batch, everything on.
        dict(name="distill_train_8192x50304", kind="distill", train=True, B=8, T=1024, V=50304, k=64, dtype="bf16", tau=2.0, weight=0.5, rest=True, hard=True, shift=False),
        # Evaluation of a student: the loss alone, teacher renormalised over its top logits.
        dict(name="distill_eval_8192x50304", kind="distill", train=False, B=8, T=1024, V=50304, k=32, dtype="bf16", tau=1.0, weight=1.0, rest=False, hard=False, shift=False),
        # fp32 logits of shifted sequences, many teacher logits.
        dict(name="distill_train_2044x32000_fp32", kind="distill", train=True, B=4, T=511, V=32000, k=256, dtype="fp32", tau=1.0, weight=0.9, rest=True, hard=True, shift=True),
        # A small ragged batch on an odd vocabulary, where latency counts.
        dict(name="distill_train_37x1003_fp16", kind="distill", train=True, B=1, T=37, V=1003, k=7, dtype="fp16", tau=4.0, weight=1.0, rest=True, hard=True, shift=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["emb", "top", "distill"], [3, 2, 3])[0]
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "emb":
        N = rng.choice([256, 512, 768, 768, 1024, 2048, 8 * rng.randint(8, 256), rng.randint(65, 1023)])
        tokens = _log(rng, 1, max(1, _MOST_EMB // N))
        B = _log(rng, 1, min(tokens, 64))
        return dict(kind=kind, train=rng.random() < 0.7, B=B, T=max(1, tokens // B), V=rng.choice([50304, 50304, 32000, 512, 1003, rng.randint(300, 60000)]), N=N,
                    dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), ids=rng.choice(["zipf", "zipf", "uniform", "one"]), scale=rng.choice([1.0, math.sqrt(N)]),
                    pad=rng.random() < 0.4)
    V = rng.choice([50304, 50304, 32000, 512, 1003, rng.randint(300, 60000)])
    rows = _log(rng, 1, _MOST // V // (2 if dtype == "fp32" else 1))
    B = _log(rng, 1, min(rows, 64))
    case = dict(kind=kind, B=B, T=max(1, rows // B), V=V, k=_log(rng, 1, 256), dtype=dtype, tau=rng.choice([1.0, 1.0, 2.0, 4.0, 0.7]), shift=rng.random() < 0.3)
    if kind == "distill":
        case.update(train=rng.random() < 0.7, weight=rng.choice([1.0, 0.5, 0.9, 0.25]), rest=rng.random() < 0.6, hard=rng.random() < 0.6)
        if not case["hard"]:
            case["weight"] = 1.0
    return case


# ---- inputs -------------------------------------------------------------------------------------


def _logits(c, g):
    """(B, T, V): near-normal logits, as a language model's are but for a few, which stand out."""
    x = torch.randn((c["B"], c["T"] + (1 if c["shift"] else 0), c["V"]), generator=g, device="cuda").mul_(2.0)
    some = torch.randint(0, c["V"], (*x.shape[:2], 4), generator=g, device="cuda")
    x.scatter_add_(-1, some, 6.0 * torch.rand(some.shape, generator=g, device="cuda"))
    return x


def _view(x, c):
    x = x.to(_DT[c["dtype"]])
    return x[:, :-1] if c["shift"] else x


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "emb":
        dt, V, shape = _DT[c["dtype"]], c["V"], (c["B"], c["T"])
        s["weight"] = (0.02 * torch.randn((V, c["N"]), generator=g, device="cuda")).to(dt).requires_grad_(c["train"])
        u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
        s["idx"] = {"zipf": lambda: (V**u).long() - 1, "uniform": lambda: (V * u).long(), "one": lambda: torch.full(shape, V // 3, device="cuda")}[c["ids"]]().clamp_(0, V - 1)
        s["pad"] = None
        if c["pad"]:  # padded sequences: the last few positions hold the padding index
            s["pad"] = V - 1
            s["idx"][:, c["T"] - c["T"] // 8 :] = V - 1
        if c["train"]:
            s["dy"] = (torch.randn((*shape, c["N"]), generator=g, device="cuda")).to(dt)
        return s
    logits = _logits(c, g)
    if c["kind"] == "top":
        s["logits"] = _view(logits, c)
        return s
    # The teacher: the student's logits and as much again of its own, its top k at the temperature kept.
    t = logits.add(torch.randn(logits.shape, generator=g, device="cuda"))
    t = t[:, :-1] if c["shift"] else t
    v, s["indices"] = torch.topk(t, c["k"], dim=-1)
    s["values"] = v.to(_DT[c["dtype"]])
    s["rest"] = None
    if c["rest"]:
        s["rest"] = t.div_(c["tau"]).scatter_(-1, s["indices"], -math.inf).logsumexp(-1)
    s["logits"] = _view(logits, c).requires_grad_(c["train"])
    s["targets"] = None
    if c["hard"]:
        targets = torch.randint(0, c["V"], (c["B"], c["T"]), generator=g, device="cuda")
        hit = torch.rand(targets.shape, generator=g, device="cuda")
        targets = torch.where(hit < 0.4, s["indices"][..., 0], targets)  # the teacher is often right
        targets = torch.where(hit > 0.9, -100, targets)  # padding
        targets[0, 0] = s["indices"][0, 0, 0]
        s["targets"] = targets
    return s


# ---- the plain forms ----------------------------------------------------------------------------


def _lse(x):
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    return (x - m).exp().sum(-1).log() + m.squeeze(-1)


def _emb(s):
    c, w, idx = s["case"], s["weight"], s["idx"]
    out = (w.detach()[idx].float() * c["scale"]).to(w.dtype)
    if not c["train"]:
        return out
    dy = s["dy"].float().view(-1, c["N"])
    if s["pad"] is not None:
        dy = dy * (idx.view(-1, 1) != s["pad"])
    dw = torch.zeros((c["V"], c["N"]), device="cuda").index_add_(0, idx.view(-1), dy)
    return out, (dw * c["scale"]).to(w.dtype)


def _top(s):
    c, x = s["case"], s["logits"]
    # One whole-number key for each logit: its order as a float, then the lower index.
    bits = (x.float() + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key = key | torch.arange(c["V"] - 1, -1, -1, device="cuda")
    indices = c["V"] - 1 - (torch.topk(key, c["k"], dim=-1).values & 0xFFFFFFFF)
    rest = _lse((x.float() / c["tau"]).scatter_(-1, indices, -math.inf))
    return x.gather(-1, indices), indices, rest


def _sums(z, tau, idx):
    """(max z, exp((z - max) / tau), the values at idx in 64 bits, their sum and the others'): a student near its teacher
    has a loss far below the logits' logsumexp, whose rounding in 32 bits would be most of it."""
    m = z.amax(-1, keepdim=True)
    e = ((z - m) / tau).exp()
    on = ((z.gather(-1, idx).double() - m) / tau).exp()
    return m, e, on, on.sum(-1, keepdim=True), e.scatter(-1, idx, 0.0).sum(-1, keepdim=True).double()


def _distill(s):
    c, k, tau, w = s["case"], s["case"]["k"], s["case"]["tau"], s["case"]["weight"]
    z, idx, targets, rest = s["logits"].detach().float(), s["indices"], s["targets"], s["rest"]
    counts = torch.ones(idx.shape[:-1], device="cuda") if targets is None else (targets != -100).float()
    n = counts.sum()
    t = s["values"].double() / tau
    if rest is not None:
        t = torch.cat((t, rest.double().unsqueeze(-1)), -1)
    logp = t - _lse(t).unsqueeze(-1)
    p = logp.exp()
    _, e, on, top, others = _sums(z, tau, idx)
    q = on / (top + others)
    classes = q if rest is None else torch.cat((q, others / (top + others)), -1)
    loss = w * tau * tau * torch.where(p > 0, p * (logp - classes.log()), 0.0).sum(-1)
    hard = targets is not None and w < 1
    if hard:
        at = targets.clamp_min(0).unsqueeze(-1)
        _, e1, on1, top1, others1 = _sums(z, 1.0, at)
        loss = loss + (1 - w) * (torch.log1p((others1 + (top1 - on1)) / on1)).squeeze(-1)
    loss = ((loss * counts).sum() / n).float()
    if not c["train"]:
        return loss
    f = 1.0 if rest is None else 1.0 - p[..., -1:] / classes[..., -1:]
    d = e.mul_((w * tau * f / (top + others)).float()).scatter_(-1, idx, (w * tau * (q - p[..., :k])).float())
    if hard:
        d.add_(e1.mul_(((1 - w) / (top1 + others1)).float())).scatter_add_(-1, at, torch.full_like(n, w - 1).expand(at.shape))
    return loss, d.mul_((counts / n).unsqueeze(-1)).to(s["logits"].dtype)


# ---- one pass -----------------------------------------------------------------------------------


@functools.cache
def _operators():
    from nanonemo_amd.kernels.hip.distill import distill_loss, top_logits
    from nanonemo_amd.kernels.hip.embedding import embedding

    return embedding, top_logits, distill_loss


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"emb": _emb, "top": _top, "distill": _distill}[c["kind"]](s)
    embedding, top_logits, distill_loss = _operators()
    if c["kind"] == "emb":
        out = embedding(s["idx"], s["weight"], scale=c["scale"], padding_idx=s["pad"])
        return (out.detach(), *torch.autograd.grad(out, s["weight"], s["dy"])) if c["train"] else out
    if c["kind"] == "top":
        return top_logits(s["logits"], c["k"], c["tau"])
    loss = distill_loss(s["logits"], s["values"], s["indices"], s["rest"], s["targets"], c["tau"], c["weight"])
    return (loss.detach(), *torch.autograd.grad(loss, s["logits"])) if c["train"] else loss


# ---- what a pass cannot do without --------------------------------------------------------------


def _rows_read(c, R):
    """The distinct rows of the weight that a batch reads, on average."""
    if c["ids"] == "one":
        return 1
    v = torch.arange(1, c["V"], dtype=torch.float64)
    p = (torch.log((v + 1) / v) / math.log(c["V"])) if c["ids"] == "zipf" else torch.full_like(v, 1 / c["V"])
    return max(1.0, float((1 - (1 - p) ** R).sum()))


def work(case):
    c, e, R = case, _SIZE[case["dtype"]], case["B"] * case["T"]
    if c["kind"] == "emb":
        rows = _rows_read(c, R)
        bytes = 8 * R + e * c["N"] * (rows + R)
        if c["train"]:
            bytes += e * c["N"] * (R + c["V"])
        return {"bytes": bytes, "flops": c["N"] * R * (3 if c["train"] else 1)}
    if c["kind"] == "top":
        return {"bytes": R * (c["V"] * e + c["k"] * (e + 8) + 4), "flops": 4 * R * c["V"]}  # compared; scaled, exp, summed
    bytes = R * (c["V"] * e + c["k"] * (e + 8) + (4 if c["rest"] else 0) + (8 if c["hard"] else 0)) + 4
    both = 2 if c["hard"] and c["weight"] < 1 and c["tau"] != 1 else 1
    flops = 3 * both * R * c["V"]
    if c["train"]:
        bytes, flops = bytes + R * c["V"] * e, 2 * flops + R * c["V"]
    return {"bytes": bytes, "flops": flops}


# ---- the same in 64 bits ------------------------------------------------------------------------


def _exact_top(s, c):
    x = s["logits"].reshape(-1, c["V"])
    values, indices, rest = [], [], []
    for part in x.split(512):
        part = part.double()
        order = torch.sort(part, dim=-1, descending=True, stable=True)
        values.append(order.values[:, : c["k"]])
        indices.append(order.indices[:, : c["k"]])
        tail = order.values[:, c["k"] :] / c["tau"]
        rest.append(tail.logsumexp(-1) if tail.shape[1] else torch.full((len(part),), -math.inf, dtype=torch.float64, device="cuda"))
    shape = s["logits"].shape[:-1]
    return torch.cat(values).view(*shape, -1), torch.cat(indices).view(*shape, -1), torch.cat(rest).view(shape)


def _exact_distill(s, c):
    """Autograd of the definition, a few hundred rows at a time."""
    V, k, R, tau, w = c["V"], c["k"], c["B"] * c["T"], c["tau"], c["weight"]
    z, v, idx = s["logits"].detach().reshape(R, V), s["values"].reshape(R, k), s["indices"].reshape(R, k)
    rest = None if s["rest"] is None else s["rest"].reshape(R, 1)
    y = None if s["targets"] is None else s["targets"].reshape(R)
    n = R if y is None else int((y != -100).sum())
    total, grads = torch.zeros((), dtype=torch.float64, device="cuda"), []
    for a in range(0, R, 512):
        b = slice(a, a + 512)
        x = z[b].double().requires_grad_()
        logq = torch.log_softmax(x / tau, -1)
        t, on = v[b].double() / tau, logq.gather(-1, idx[b])
        if rest is not None:
            t = torch.cat((t, rest[b].double()), -1)
            others = torch.ones_like(logq, dtype=torch.bool).scatter_(-1, idx[b], False)
            on = torch.cat((on, logq.masked_fill(~others, -math.inf).logsumexp(-1, keepdim=True)), -1)
        p = torch.softmax(t, -1)
        row = w * tau**2 * torch.special.xlogy(p, p).sub(torch.where(p > 0, p * on, 0.0)).sum(-1)
        if y is not None:
            keep = y[b] != -100
            if w < 1:
                row = row - (1 - w) * torch.log_softmax(x, -1).gather(-1, y[b].clamp_min(0).unsqueeze(-1)).squeeze(-1)
            row = torch.where(keep, row, 0.0)
        part = row.sum() / n
        total += part.detach()
        if c["train"]:
            grads.append(torch.autograd.grad(part, x)[0])
    return (total, torch.cat(grads).view(s["logits"].shape)) if c["train"] else total


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "top":
        return _exact_top(s, c)
    if c["kind"] == "distill":
        return _exact_distill(s, c)
    w, idx = s["weight"].detach().double(), s["idx"].reshape(-1)
    out = (w.index_select(0, idx) * c["scale"]).view(c["B"], c["T"], c["N"])
    if not c["train"]:
        return out
    order = torch.argsort(idx, stable=True)  # the tokens of each row of the weight side by side: differences of a running sum
    run = s["dy"].reshape(-1, c["N"]).double().mul(c["scale"])[order].cumsum(0)
    ids, last = torch.unique_consecutive(idx[order], return_counts=True)
    ends = run[last.cumsum(0) - 1]
    dw = torch.zeros_like(w)
    dw[ids] = ends - torch.cat((torch.zeros_like(ends[:1]), ends[:-1]))
    if s["pad"] is not None:
        dw[s["pad"]] = 0
    return out, dw
