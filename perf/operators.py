"""The objectives over logits (rustautograd_b200.losses) as measured cases: the log-probability of given
tokens, the clipped policy loss with a KL term, the preference loss over pairs of sequences and the
distillation from a teacher's top logits, each with its gradient.

`run` gives each operator's outputs in its plain form (elementary torch operations) or, with `own`, through
the calls a program makes on arrays that are already in device memory.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f64": torch.float64}
CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def listed():
    """Sequences x length x vocabulary. `shift`: the logits are the first `length` positions of a model's output
    of length + 1 (next-token prediction), a strided view. `pad`: the share of positions behind the sequences'
    ends (weight 0, labels of -100, logits of any value). `ban`: columns whose logits are -inf."""
    return [
        # One sampled token of each of 8 running sequences, scored: only latency counts.
        {"name": "logprob_step", "op": "logprob", "n": 8, "t": 1, "v": 32000, "dtype": "f32", "shift": False, "ban": 0, "grad": False},
        # Old or reference log-probabilities of a batch of samples, odd vocabulary.
        {"name": "logprob_batch", "op": "logprob", "n": 16, "t": 511, "v": 50257, "dtype": "f32", "shift": True, "ban": 37, "grad": False},
        # A double-precision check of a training step: forward and gradient, all sizes odd.
        {"name": "logprob_train_f64", "op": "logprob", "n": 3, "t": 341, "v": 4093, "dtype": "f64", "shift": False, "ban": 0, "grad": True},
        # The character GPT of the repository's benchmark (batch 512, context 256, vocabulary 96).
        {"name": "policy_char", "op": "policy", "n": 512, "t": 256, "v": 96, "dtype": "f32", "shift": False, "ban": 0, "pad": 0.1, "kl": 0.0, "grad": True},
        # A small step of a few short answers.
        {"name": "policy_small", "op": "policy", "n": 4, "t": 61, "v": 32000, "dtype": "f32", "shift": True, "ban": 0, "pad": 0.2, "kl": 0.02, "grad": True},
        # The largest: a full batch of long answers, odd vocabulary, constrained decoding, KL to the reference.
        {"name": "policy_large", "op": "policy", "n": 16, "t": 1024, "v": 50257, "dtype": "f32", "shift": True, "ban": 101, "pad": 0.15, "kl": 0.02, "grad": True},
        # The loss alone, watched on held-out samples in double precision.
        {"name": "policy_eval_f64", "op": "policy", "n": 7, "t": 129, "v": 10007, "dtype": "f64", "shift": False, "ban": 5, "pad": 0.3, "kl": 0.1, "grad": False},
        # Two pairs of short sequences.
        {"name": "preference_small", "op": "preference", "n": 4, "t": 37, "v": 1009, "dtype": "f32", "shift": True, "ban": 0, "pad": 0.3, "smooth": 0.1, "grad": True},
        # Eight pairs, prompts and padding masked.
        {"name": "preference", "op": "preference", "n": 16, "t": 512, "v": 32000, "dtype": "f32", "shift": True, "ban": 11, "pad": 0.25, "smooth": 0.0, "grad": True},
        # A small distillation step.
        {"name": "distill_small", "op": "distill", "n": 2, "t": 24, "v": 50257, "dtype": "f32", "shift": False, "ban": 0, "pad": 0.1, "k": 8, "temp": 1.0, "grad": True},
        # A full distillation batch over a long vocabulary.
        {"name": "distill", "op": "distill", "n": 4, "t": 1024, "v": 131072, "dtype": "f32", "shift": False, "ban": 0, "pad": 0.1, "k": 64, "temp": 2.0, "grad": True},
        # The loss alone on held-out text.
        {"name": "distill_eval", "op": "distill", "n": 5, "t": 203, "v": 8191, "dtype": "f32", "shift": True, "ban": 7, "pad": 0.2, "k": 20, "temp": 1.5, "grad": False},
    ]


def draw(rng):
    def log_uniform(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["logprob", "policy", "preference", "distill"])
    dtype = "f64" if rng.random() < 0.2 else "f32"
    c = {"op": op, "dtype": dtype, "grad": rng.random() < 0.75, "shift": rng.random() < 0.5}
    c["v"] = log_uniform(65, 150000)
    most = 300_000_000 // c["v"] // (2 if dtype == "f64" else 1)  # rows: at most 1.2 GB of logits
    c["n"] = log_uniform(1, max(1, min(512, most // 4)))
    if op == "preference":
        c["n"] = max(2, c["n"] // 2 * 2)
    c["t"] = log_uniform(1, max(1, min(2048, most // c["n"])))
    c["ban"] = rng.choice([0, 0, c["v"] // 50])
    if op != "logprob":
        c["pad"] = rng.choice([0.0, 0.1, 0.4])
    if op == "policy":
        c["kl"] = rng.choice([0.0, 0.02, 0.1])
    if op == "preference":
        c["smooth"] = rng.choice([0.0, 0.1])
    if op == "distill":
        c["k"] = min(c["v"], log_uniform(1, 128))
        c["temp"] = rng.choice([1.0, 1.5, 2.0])
    return c


def _lengths(case):
    """Sequence lengths with the case's share of padding: spread evenly, the same total for every seed."""
    n, t, pad = case["n"], case["t"], case.get("pad", 0.0)
    return [t - int(2 * pad * t * b / max(1, n - 1)) if n > 1 else t for b in range(n)]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    n, t, v, dt = case["n"], case["t"], case["v"], DTYPES[case["dtype"]]
    dev = "cuda"

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=g, device=dev, dtype=dt) * (hi - lo) + lo

    full = torch.randn((n, t + 1 if case["shift"] else t, v), generator=g, device=dev, dtype=dt).mul_(2.5)
    logits = full[:, :t]
    labels = torch.randint(0, v, (n, t), generator=g, device=dev, dtype=torch.int32)
    if case["ban"]:
        banned = torch.randint(0, v, (case["ban"],), generator=g, device=dev)
        full[..., banned] = -math.inf
    # The label's logit: from unlikely tokens to nearly certain ones.
    logits.scatter_(2, labels.long()[..., None], uniform(4.0, 7.0 + math.log(v), n, t, 1))
    s = {"case": case, "logits": logits, "labels": labels}
    if case["op"] == "logprob":
        s["dlogp"] = uniform(-1.0, 1.0, n, t) / (n * t)
        return s
    lengths = torch.tensor(random.Random(seed).sample(_lengths(case), n), device=dev)
    mask = torch.arange(t, device=dev)[None, :] < lengths[:, None]
    if case["op"] == "policy":
        logp = torch.log_softmax(logits, -1).gather(2, labels.long()[..., None])[..., 0]
        # The probability ratio, drawn as a few updates after the sampling leave it. Ratios within 0.002 of a clip
        # bound are moved off it: which side of the bound such a token falls on is up to its last bits.
        ratio = torch.exp(torch.randn((n, t), generator=g, device=dev, dtype=dt) * 0.2)
        for edge in (1.0 - CLIP_LOW, 1.0 + CLIP_HIGH):
            ratio = torch.where((ratio - edge).abs() < 0.002, torch.full_like(ratio, edge + 0.004), ratio)
        s["old"] = logp - ratio.log()
        s["advantage"] = torch.randn((n, t), generator=g, device=dev, dtype=dt)
        s["weight"] = mask.to(dt) / mask.sum().to(dt)
        if case["kl"]:
            s["ref"] = logp + torch.randn((n, t), generator=g, device=dev, dtype=dt) * 0.3
    if case["op"] == "preference":
        prompt = torch.arange(t, device=dev)[None, :] >= t // 8  # the prompt's own tokens do not count
        s["weight"] = (mask & prompt).to(dt)
        logp = torch.log_softmax(logits, -1).gather(2, labels.long()[..., None])[..., 0]
        s["ref"] = torch.where(mask & prompt, logp, 0).sum(1) + torch.randn((n,), generator=g, device=dev, dtype=dt) * 8.0
    if case["op"] == "distill":
        k = case["k"]
        # The teacher's likeliest tokens are likely under the student too, and never banned ones.
        s["index"] = torch.randint(0, v, (n, t, k), generator=g, device=dev, dtype=torch.int32)
        at = s["index"].long()
        logits.scatter_(2, at, uniform(2.0, 9.0, v)[at])
        teacher = torch.sort(uniform(0.0, 9.0, n, t, k), -1, descending=True).values
        some = torch.rand((n, t, 1), generator=g, device=dev) < 0.1  # rows that hold fewer than k entries
        s["teacher"] = torch.where(some & (torch.arange(k, device=dev) >= max(1, k // 2)), -math.inf, teacher)
        s["weight"] = mask.to(dt) / mask.sum().to(dt)
    # What a batch holds behind its sequences' ends: labels that name nothing, logits that may be anything.
    if case.get("pad"):
        s["labels"] = torch.where(mask, labels, -100)
        behind = (~mask).nonzero()[:4096:7]
        logits[behind[:, 0], behind[:, 1]] = math.nan
    return s


def run(s):
    if own:
        return _own(s)
    return {"logprob": _logprob, "policy": _policy, "preference": _preference, "distill": _distill}[s["case"]["op"]](s)


def _own(s):
    from rustautograd_b200 import losses

    c, grad = s["case"], s["case"]["grad"]
    if c["op"] == "logprob":
        if not grad:
            return losses.token_log_prob(s["logits"], s["labels"])
        logp, stats = losses.token_log_prob(s["logits"], s["labels"], stats=True)
        return logp, losses.token_log_prob_grad(s["logits"], s["labels"], stats, s["dlogp"])
    if c["op"] == "policy":
        r = losses.policy_loss(s["logits"], s["labels"], s["old"], s["advantage"], s["weight"], ref_logp=s.get("ref"),
                               clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl=c["kl"], grad=grad)
        return r.loss, r.logp, r.grad
    if c["op"] == "preference":
        r = losses.preference_loss(s["logits"], s["labels"], s["weight"], s["ref"], beta=0.1, smoothing=c["smooth"], grad=grad)
        return r.loss, r.margins, r.logp, r.grad
    r = losses.distillation_loss(s["logits"], s["index"], s["teacher"], s["weight"], temperature=c["temp"], grad=grad)
    return r.loss, r.terms, r.grad


# ---- plain forms ----

def _softmax(x):
    """(row max, sum of exp(x - max), softmax) along the last axis."""
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    return m, z, e.div_(z)


def _picked(x, m, z, labels):
    at = labels.clamp(0, x.shape[-1] - 1).long()[..., None]
    return (x.gather(-1, at) - m - torch.log(z))[..., 0], at


def _logprob(s):
    x = s["logits"]
    m, z, p = _softmax(x)
    logp, at = _picked(x, m, z, s["labels"])
    if not s["case"]["grad"]:
        return logp
    c = s["dlogp"][..., None]
    return logp, p.mul_(-c).scatter_add_(-1, at, c)


def _rows(live, x):
    """Rows without weight as zeros, whatever they hold."""
    return torch.where(live[..., None], x, 0)


def _policy(s):
    x, w, a, kl = s["logits"], s["weight"], s["advantage"], s["case"]["kl"]
    live = w != 0
    m, z, p = _softmax(x)
    logp, at = _picked(x, m, z, s["labels"])
    logp = torch.where(live, logp, 0)
    ratio = torch.exp(logp - s["old"])
    term = -torch.minimum(ratio * a, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * a)
    active = torch.where(a >= 0, ratio <= 1.0 + CLIP_HIGH, ratio >= 1.0 - CLIP_LOW)
    c = torch.where(active, -a * ratio, 0)
    if kl:
        d = s["ref"] - logp
        term = term + kl * (torch.exp(d) - d - 1.0)
        c = c + kl * (1.0 - torch.exp(d))
    loss = torch.where(live, w * term, 0).double().sum().to(x.dtype)
    c = torch.where(live, w * c, 0)[..., None]
    return loss, logp, _rows(live, p.mul_(-c).scatter_add_(-1, at, c)) if s["case"]["grad"] else None


def _preference(s):
    x, w, n, eps, beta = s["logits"], s["weight"], s["case"]["n"] // 2, s["case"]["smooth"], 0.1
    live = w != 0
    m, z, p = _softmax(x)
    logp, at = _picked(x, m, z, s["labels"])
    total = torch.where(live, w * logp, 0).double().sum(-1)
    gain = total - s["ref"].double()
    h = beta * (gain[:n] - gain[n:])
    up, down = 1.0 / (1.0 + torch.exp(-h)), 1.0 / (1.0 + torch.exp(h))
    softplus = torch.log1p(torch.exp(-h.abs()))
    loss = ((1.0 - eps) * (softplus + (-h).clamp(min=0)) + eps * (softplus + h.clamp(min=0))).mean()
    dh = (eps * up - (1.0 - eps) * down) / n
    c = (torch.cat([dh, -dh])[:, None] * beta * w).to(x.dtype)[..., None]
    grad = _rows(live, p.mul_(-c).scatter_add_(-1, at, c)) if s["case"]["grad"] else None
    return loss.to(x.dtype), h.to(x.dtype), total.to(x.dtype), grad


def _distill(s):
    x, w, t = s["logits"], s["weight"], s["case"]["temp"]
    at = s["index"].long()
    q = _softmax(s["teacher"] / t)[2]
    m, z, p = _softmax(x / t)
    logp = x.gather(-1, at) / t - m - torch.log(z)
    live = w != 0
    term = torch.where(live, w * t * t * torch.where(q > 0, q * (torch.log(q) - logp), 0).sum(-1), 0)
    loss = term.double().sum().to(x.dtype)
    if not s["case"]["grad"]:
        return loss, term, None
    c = (w * t)[..., None]
    return loss, term, _rows(live, p.mul_(c).scatter_add_(-1, at, -c * q))


def exact(case, seed):
    """The same outputs from the definitions in 64 bits."""
    s = prepare(case, seed)
    x, op, grad = s["logits"].double(), case["op"], case["grad"]
    v = x.shape[-1]
    onehot_at = s["labels"].long().clamp(0, v - 1).unsqueeze(-1)
    if op == "logprob":
        logp = x.gather(-1, onehot_at).squeeze(-1) - torch.logsumexp(x, -1)
        if not grad:
            return logp
        d = s["dlogp"].double().unsqueeze(-1)
        g = torch.softmax(x, -1) * -d
        return logp, g.scatter_add(-1, onehot_at, d)
    w = s["weight"].double()
    keep = (w != 0).unsqueeze(-1)
    x = torch.where(keep, x, torch.zeros((), dtype=x.dtype, device=x.device))
    if op == "distill":
        t, at = case["temp"], s["index"].long()
        logq = torch.log_softmax(s["teacher"].double() / t, -1)
        q = logq.exp()
        logp = torch.log_softmax(x / t, -1)
        kl = torch.where(q == 0, torch.zeros_like(q), q * (logq - logp.gather(-1, at))).sum(-1)
        term = w * t * t * kl
        if not grad:
            return term.sum(), term, None
        g = logp.exp_().scatter_add_(-1, at, -q) * (w * t).unsqueeze(-1)
        return term.sum(), term, g
    logp = x.gather(-1, onehot_at).squeeze(-1) - torch.logsumexp(x, -1)
    if op == "policy":
        logp = torch.where(w != 0, logp, torch.zeros_like(logp))
        a = s["advantage"].double()
        r = torch.exp(logp - s["old"].double())
        inside = torch.clamp(r, 1 - CLIP_LOW, 1 + CLIP_HIGH)
        term = torch.where(w != 0, -torch.minimum(r * a, inside * a), torch.zeros_like(r))
        slope = torch.where(r * a <= inside * a, -r * a, torch.zeros_like(r))
        if case["kl"]:
            d = s["ref"].double() - logp
            term = term + case["kl"] * torch.where(w != 0, torch.expm1(d) - d, torch.zeros_like(d))
            slope = slope - case["kl"] * torch.expm1(d)
        head = ((w * term).sum(), logp)
        c = torch.where(w != 0, w * slope, torch.zeros_like(w))
    else:
        n, eps = case["n"] // 2, case["smooth"]
        total = (w * logp).sum(-1)
        gain = total - s["ref"].double()
        h = 0.1 * (gain[:n] - gain[n:])
        loss = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h)).mean()
        slope = -((1 - eps) - torch.sigmoid(h)) / n
        head = (loss, h, total)
        c = torch.cat([slope, -slope]).unsqueeze(-1) * 0.1 * w
    if not grad:
        return (*head, None)
    c = c.unsqueeze(-1)
    return (*head, (torch.softmax(x, -1) * -c).scatter_add_(-1, onehot_at, c))


def work(case):
    """The logits read once and, where asked for, their gradient written once; rows without weight need no reading."""
    size = 8 if case["dtype"] == "f64" else 4
    rows, v = case["n"] * case["t"], case["v"]
    live = sum(_lengths(case)) if case["op"] in ("policy", "distill") else rows
    if case["op"] == "preference":
        live = sum(max(0, length - case["t"] // 8) for length in _lengths(case))
    per_row = {"logprob": 4 + 3 * size, "policy": 4 + 5 * size, "preference": 4 + size, "distill": case.get("k", 0) * (4 + size) + 2 * size}[case["op"]]
    return {"bytes": live * v * size + (rows * v * size if case["grad"] else 0) + rows * per_row, "flops": live * v * (7 if case["grad"] else 4)}
