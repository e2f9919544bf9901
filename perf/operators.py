"""What is measured of the vocabulary-row operators, and their plain forms.

Three operators over rows of logits z[row][vocab] at a temperature T, with
p = softmax(z / T) of the row:

* score:       log p of given tokens, the entropy of p, the top_k alternatives
               (ids by logit descending, equal logits by ascending id) and their log p
* score_grad:  the gradient of sum(g_logprob * log p[token]) + sum(g_entropy * entropy)
               with respect to the logits
* distill:     per row (1 - a) T^2 KL(q || p) + a (-log softmax(z)[label]) against a
               teacher's top logits (ids, values): q is the softmax of the listed values
               over T; with `rest` the values are log probabilities already at T, and
               what they leave of 1 is one more outcome, matched with the student's mass
               outside the list.  And the gradient of sum(row_grad * loss).

Ids outside the vocabulary are padding: they give log p 0, carry no teacher
mass and no gradient.  A logit of -inf is masked: its gradient is 0.

`own` false computes them with elementary torch operations in 32 bits; `own`
true through this package's entry points.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ESIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
MOST = 2048 * 131072  # logits of the largest case


def _score(name, rows, vocab, dtype, top_k, temperature=1.0, n_tok=1, masked=0.0, pad=0, spread=2.5):
    return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "temperature": temperature, "n_tok": n_tok, "masked": masked, "pad": pad, "spread": spread}


def _grad(name, rows, vocab, dtype, temperature=1.0, n_tok=1, entropy=True, masked=0.0, pad=0, spread=2.5):
    return {"name": name, "op": "score_grad", "rows": rows, "vocab": vocab, "dtype": dtype, "entropy": entropy,
            "temperature": temperature, "n_tok": n_tok, "masked": masked, "pad": pad, "spread": spread}


def _distill(name, rows, vocab, dtype, top_k, temperature=1.0, label_weight=0.0, rest=False, grad=True, masked=0.0,
             pad=0, spread=2.5):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "temperature": temperature, "label_weight": label_weight, "rest": rest, "grad": grad, "masked": masked,
            "pad": pad, "spread": spread}


def listed():
    return [
        # one sequence's decode step, its token's log probability shown with 20 alternatives: latency
        _score("score_one_row", 1, 16384, "fp32", 20, spread=4.0),
        # a decode step of 512 sequences under the sampling temperature, with alternatives
        _score("score_512_v16384", 512, 16384, "fp32", 20, temperature=0.7),
        # a long text's perplexity and entropy, no alternatives: half-precision logits, a vocabulary of 32000
        _score("score_8192_v32000_bf16", 8192, 32000, "bf16", 0),
        # a teacher's top logits for distillation over a large vocabulary
        _score("score_teacher_v131072", 2048, 131072, "fp32", 64, temperature=2.0),
        # constrained decoding: a tenth of an odd vocabulary masked, rows not 16-byte aligned, four tokens a row
        _score("score_masked_v50001", 301, 50001, "fp16", 128, n_tok=4, masked=0.1, pad=3),
        # policy gradient with an entropy bonus over one sequence of 1024 tokens
        _grad("grad_1024_v16384", 1024, 16384, "fp32"),
        # log-probability gradient of a batch at a large vocabulary, half precision
        _grad("grad_2048_v131072_bf16", 2048, 131072, "bf16", entropy=False),
        # few rows, an odd small vocabulary, several tokens a row
        _grad("grad_33_v1001", 33, 1001, "fp32", temperature=0.7, n_tok=3, masked=0.1),
        # the training step's shape: one sequence of 1024 positions, 64 teacher logits, half the loss from the labels
        _distill("distill_1024_v16384", 1024, 16384, "fp32", 64, temperature=2.0, label_weight=0.5),
        # a batch in half precision with the rest of the vocabulary as one outcome
        _distill("distill_rest_4096_v32000_bf16", 4096, 32000, "bf16", 128, rest=True),
        # the largest vocabulary, the teacher's top 20 of a served model, the rest as one outcome
        _distill("distill_rest_2048_v131072", 2048, 131072, "fp32", 20, temperature=1.5, rest=True),
        # evaluation of a small student: the loss alone, rows not 16-byte aligned
        _distill("distill_loss_97_v16383", 97, 16383, "fp32", 32, temperature=2.0, grad=False, pad=2),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "score_grad", "distill"])
    vocab = _log_int(rng, 256, 131072)
    if rng.random() < 0.5:
        vocab -= vocab % 8  # vocabularies are often padded to a multiple of 8
    rows = min(_log_int(rng, 1, 8192), MOST // vocab)
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
            "temperature": rng.choice([1.0, round(rng.uniform(0.3, 3.0), 3)]),
            "masked": rng.choice([0.0, 0.0, 0.1, 0.5]), "pad": rng.choice([0, 0, 8, rng.randrange(1, 8)]),
            "spread": round(rng.uniform(1.0, 4.0), 2)}
    if op == "score":
        case |= {"top_k": rng.choice([0, _log_int(rng, 1, 512)]), "n_tok": rng.choice([1, 1, _log_int(rng, 2, 64)])}
        case["top_k"] = min(case["top_k"], vocab)
    elif op == "score_grad":
        case |= {"n_tok": rng.choice([1, 1, _log_int(rng, 2, 64)]), "entropy": rng.random() < 0.5}
    else:
        case |= {"top_k": min(_log_int(rng, 1, 512), vocab // 2), "label_weight": rng.choice([0.0, 0.3, 0.5]),
                 "rest": rng.random() < 0.5, "grad": rng.random() < 0.75}
    return case


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rows, vocab, T = case["rows"], case["vocab"], case["temperature"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    # a model's logits: a bulk of the given spread and a few likely tokens far above it
    x = randn(rows, vocab).mul_(case["spread"])
    likely = torch.randint(0, vocab // 8, (rows, 8), generator=g, device=dev)
    likely += vocab // 8 * torch.arange(8, device=dev)  # eight different ones
    x.scatter_add_(1, likely, 10.0 * rand(rows, 8))
    s = dict(case)
    if case["op"] == "distill":
        # the teacher: another model's logits of the same text
        t = (x + 0.7 * randn(rows, vocab)) / T
        if case["rest"]:
            t -= torch.logsumexp(t, 1, keepdim=True)
        else:
            t *= T
        val, ids = torch.topk(t, case["top_k"], dim=1)
        del t
        used = torch.randint(1 + 3 * case["top_k"] // 4, case["top_k"] + 1, (rows, 1), generator=g, device=dev) \
            if case["top_k"] >= 4 else torch.full((rows, 1), case["top_k"], device=dev)
        ids = torch.where(torch.arange(case["top_k"], device=dev) < used, ids, -1)  # lists of unequal length
        ids[rand(rows) < 0.05] = -1  # rows past the end of a text
        s["teacher_ids"], s["teacher_logits"] = ids.int(), val.float()
        labels = likely[:, 0].clone()
        labels[rand(rows) < 0.05] = -1
        s["labels"] = labels.int() if case["label_weight"] > 0 else None
        s["row_grad"] = 0.5 + rand(rows)  # weights of a loss summed over the rows
        keep = torch.cat([ids.clamp(min=0).long(), likely[:, :1]], 1)
    else:
        n = case["n_tok"]
        tokens = torch.randint(0, vocab, (rows, n), generator=g, device=dev)
        tokens[:, : min(n, 8)] = likely[:, : min(n, 8)]
        keep = tokens
        s["tokens"] = torch.where(rand(rows, 1) < 0.05, -1, tokens).int()
        if n == 1:
            s["tokens"] = s["tokens"][:, 0].contiguous()
        if case["op"] == "score_grad":
            s["g_logprob"] = randn(*s["tokens"].shape)
            s["g_entropy"] = 0.01 * rand(rows) if case["entropy"] else None
    if case["masked"]:
        off = rand(rows, vocab) < case["masked"]
        off.scatter_(1, keep, False)
        x.masked_fill_(off, -math.inf)
    out = torch.empty(rows, vocab + case["pad"], dtype=DTYPES[case["dtype"]], device=dev)
    out.fill_(0.0)
    out[:, :vocab] = x
    s["logits"] = out[:, :vocab]
    return s


# ---- the plain forms: elementary operations in 32 bits ----

def _log_p(logits, T):
    x = logits.float()
    x = (x - x.amax(1, keepdim=True)) / T
    return x - torch.log(torch.exp(x).sum(1, keepdim=True))


def _at(x, ids):
    """x[row][ids] with 0 where an id is padding."""
    v = torch.gather(x, 1, ids.clamp(min=0).long())
    return torch.where(ids >= 0, v, 0.0)


def _plain_score(s):
    logits, vocab = s["logits"], s["vocab"]
    lp = _log_p(logits, s["temperature"])
    tok = s["tokens"].view(s["rows"], -1)
    out = {"logprob": _at(lp, tok).view(s["tokens"].shape)}
    p = torch.exp(lp)
    out["entropy"] = -torch.where(p > 0, p * lp, 0.0).sum(1)
    if s["top_k"]:
        # descending logits, equal ones by ascending id, as one 64-bit key an entry
        b = (logits.float() + 0.0).view(torch.int32)
        key = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long() * (1 << 32)
        key += vocab - 1 - torch.arange(vocab, device=key.device)
        top = torch.topk(key, s["top_k"], dim=1).values
        ids = vocab - 1 - (top & 0xFFFFFFFF)
        out["top_ids"] = ids.int()
        out["top_logprob"] = torch.gather(lp, 1, ids)
    return out


def _plain_score_grad(s):
    logits, T = s["logits"], s["temperature"]
    lp = _log_p(logits, T)
    p = torch.exp(lp)
    tok = s["tokens"].view(s["rows"], -1)
    g = torch.where(tok >= 0, s["g_logprob"].view(tok.shape), 0.0)
    d = p * -g.sum(1, keepdim=True)
    d.scatter_add_(1, tok.clamp(min=0).long(), g)
    if s["g_entropy"] is not None:
        plp = torch.where(p > 0, p * lp, 0.0)
        ent = -plp.sum(1, keepdim=True)
        d -= s["g_entropy"][:, None] * (plp + p * ent)
    d = torch.where(logits == -math.inf, 0.0, d / T)
    return {"grad": d.to(logits.dtype)}


def _plain_distill(s):
    logits, T, a = s["logits"], s["temperature"], s["label_weight"]
    rows, vocab = logits.shape
    ids = s["teacher_ids"].long()
    valid = ids >= 0
    some = valid.any(1)
    col = torch.where(valid, ids, vocab)  # padding goes to a column behind the vocabulary
    x = logits.float()
    x = torch.cat([(x - x.amax(1, keepdim=True)) / T, torch.zeros_like(x[:, :1])], 1)
    e = torch.exp(x)
    e[:, vocab] = 0.0
    # a row's scalars in 64 bits: long sums, and a loss that is a small difference of large terms
    total = e.sum(1, dtype=torch.float64)
    lq = torch.where(valid, s["teacher_logits"], -math.inf).double()
    if not s["rest"]:
        lq = lq / T
        lq = lq - torch.where(some, lq.amax(1), 0.0)[:, None]
        lq = lq - torch.log(torch.exp(lq).sum(1, keepdim=True))
        lq = torch.where(valid, lq, -math.inf)
    q = torch.exp(lq)
    lp = torch.gather(x, 1, col).double() - torch.log(total)[:, None]
    loss = torch.where(q > 0, q * (lq - lp), 0.0).sum(1)
    mass = q.sum(1)
    if s["rest"]:
        # what the list leaves: 1 - sum q for the teacher, the unlisted sum for the student
        r = torch.where(some, (1.0 - mass).clamp(min=0), 0.0)
        rest = e.scatter(1, col, 0.0)
        u = rest.sum(1, dtype=torch.float64) / total
        r = torch.where(u > 0, r, 0.0)
        loss = loss + torch.where(r > 0, r * (torch.log(r) - torch.log(u)), 0.0)
        mass = mass + r
    loss = loss * ((1 - a) * T * T)
    d = None
    if s["grad"]:
        d = e * (mass / total).float()[:, None]
        if s["rest"]:
            d = d - rest * torch.where(r > 0, r / (u * total), 0.0).float()[:, None]
        d.scatter_add_(1, col, -q.float())
        d = d[:, :vocab] * ((1 - a) * T)
    if s["labels"] is not None:
        y = s["labels"].view(-1, 1)
        l1 = _log_p(logits, 1.0)
        loss = loss - a * _at(l1, y)[:, 0]
        if s["grad"]:
            on = torch.where(y >= 0, a, 0.0)
            d = d + torch.exp(l1) * on
            d.scatter_add_(1, y.clamp(min=0).long(), -on)
    loss = loss.float()
    out = {"loss": loss}
    if s["grad"]:
        d = torch.where(logits == -math.inf, 0.0, d * s["row_grad"][:, None])
        out["grad"] = d.to(logits.dtype)
    return out


def run(s):
    op = s["op"]
    if own:
        import snai_b200 as sn
        if op == "score":
            r = sn.score_device(s["logits"], s["tokens"], temperature=s["temperature"], top_k=s["top_k"])
            out = {"logprob": r.logprob, "entropy": r.entropy}
            if s["top_k"]:
                out |= {"top_ids": r.top_ids, "top_logprob": r.top_logprob}
            return out
        if op == "score_grad":
            return {"grad": sn.score_grad_device(s["logits"], s["tokens"], s["g_logprob"], s["g_entropy"],
                                                 temperature=s["temperature"])}
        loss, grad = sn.distill_device(s["logits"], s["teacher_ids"], s["teacher_logits"], labels=s["labels"],
                                       temperature=s["temperature"], label_weight=s["label_weight"],
                                       rest=s["rest"], row_grad=s["row_grad"], want_grad=s["grad"])
        return {"loss": loss, "grad": grad} if s["grad"] else {"loss": loss}
    return {"score": _plain_score, "score_grad": _plain_score_grad, "distill": _plain_distill}[op](s)


def work(case):
    rows, vocab, e = case["rows"], case["vocab"], ESIZE[case["dtype"]]
    n = rows * vocab
    if case["op"] == "score":
        # logits in; token ids in and their log p out; entropies out; (id, log p) of the alternatives out
        return {"bytes": n * e + rows * (8 * case["n_tok"] + 4 + 8 * case["top_k"]), "flops": 6 * n}
    if case["op"] == "score_grad":
        # logits in, gradient out; token ids and their gradients in
        return {"bytes": 2 * n * e + rows * (8 * case["n_tok"] + 4 * case["entropy"]), "flops": 10 * n}
    small = rows * (8 * case["top_k"] + 4 + (4 if case["label_weight"] > 0 else 0) + (4 if case["grad"] else 0))
    return {"bytes": (2 if case["grad"] else 1) * n * e + small, "flops": (8 if case["grad"] else 5) * n}


# ---- the definition in 64 bits, a block of rows at a time ----

def _exact_score(s, lo, hi):
    z = s["logits"][lo:hi].double() / s["temperature"]
    lse = torch.logsumexp(z, 1)
    tok = s["tokens"][lo:hi].long()
    t2 = tok.reshape(hi - lo, -1)
    lp = z.gather(1, t2.clamp_min(0)) - lse[:, None]
    mean = (torch.softmax(z, 1) * z.masked_fill(z == -math.inf, 0.0)).sum(1)
    out = {"logprob": lp.masked_fill(t2 < 0, 0.0).reshape(tok.shape), "entropy": lse - mean}
    if s["top_k"]:
        out |= {"top_ids": None, "top_logprob": z.topk(s["top_k"], 1).values - lse[:, None]}
    return out


def _exact_score_grad(s, lo, hi):
    T = s["temperature"]
    z = s["logits"][lo:hi].double()
    p = torch.softmax(z / T, 1)
    tok = s["tokens"][lo:hi].long().reshape(hi - lo, -1)
    g = s["g_logprob"][lo:hi].double().reshape(tok.shape) * (tok >= 0)
    hot = torch.zeros_like(p).scatter_add_(1, tok.clamp_min(0), g)
    d = hot - p * g.sum(1, keepdim=True)
    if s["g_entropy"] is not None:
        zf = (z / T).masked_fill(z == -math.inf, 0.0)
        mean = (p * zf).sum(1, keepdim=True)  # dH/dz = -p (z - E z) / T, with z over T
        d = d - s["g_entropy"][lo:hi].double()[:, None] * p * (zf - mean)
    return {"grad": (d / T).masked_fill(z == -math.inf, 0.0)}


def _exact_distill(s, lo, hi):
    T, a = s["temperature"], s["label_weight"]
    z = s["logits"][lo:hi].double()
    R, V = z.shape
    ids, t = s["teacher_ids"][lo:hi].long(), s["teacher_logits"][lo:hi].double()
    ok = ids >= 0
    q = torch.exp(t) if s["rest"] else torch.exp(t / T)
    q = q * ok
    if not s["rest"]:
        q = q / q.sum(1, keepdim=True).masked_fill(~ok.any(1, keepdim=True), 1.0)
    dense = torch.zeros(R, V, dtype=torch.float64, device=z.device).scatter_add_(1, ids.clamp_min(0), q)
    on = torch.zeros(R, V, dtype=torch.int32, device=z.device).scatter_add_(1, ids.clamp_min(0), ok.int()) > 0
    logp = torch.log_softmax(z / T, 1)
    p = logp.exp()
    loss = torch.special.xlogy(q, q).sum(1) - (dense * logp.masked_fill(~on, 0.0)).sum(1)
    target = dense
    if s["rest"]:
        r = (1.0 - q.sum(1)).clamp_min(0.0) * ok.any(1)
        u = (p * ~on).sum(1)
        r = r * (u > 0)
        loss = loss + torch.special.xlogy(r, r) - torch.special.xlogy(r, u.masked_fill(u <= 0, 1.0))
        share = (r / u.masked_fill(u <= 0, 1.0))[:, None]
        target = dense + (p * ~on) * share  # the rest's mass, spread as the student spreads its own
    d = (p * target.sum(1, keepdim=True) - target) * ((1 - a) * T)
    loss = loss * ((1 - a) * T * T)
    if s["labels"] is not None:
        y = s["labels"][lo:hi].long()
        l1 = torch.log_softmax(z, 1)
        w = a * (y >= 0).double()
        loss = loss - w * l1.gather(1, y.clamp_min(0)[:, None])[:, 0]
        d = d + w[:, None] * l1.exp()
        d.scatter_add_(1, y.clamp_min(0)[:, None], -w[:, None])
    out = {"loss": loss}
    if s["grad"]:
        out["grad"] = (d * s["row_grad"][lo:hi].double()[:, None]).masked_fill(z == -math.inf, 0.0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    f = {"score": _exact_score, "score_grad": _exact_score_grad, "distill": _exact_distill}[s["op"]]
    step = max(1, (1 << 26) // s["vocab"])
    parts = [f(s, lo, min(lo + step, s["rows"])) for lo in range(0, s["rows"], step)]
    return {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts]) for k in parts[0]}
