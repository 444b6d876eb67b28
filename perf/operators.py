"""Measured cases of the language-model operators: embedding lookup and its gradient, the gated linear recurrence
and its gradient, log probabilities of given tokens with entropy and top alternatives and their gradient.

``run`` computes a case either in plain form (elementary torch operations in float32, rounded once at the end) or,
where ``own`` is true, with this package's entry points.  ``exact`` computes the same from the definitions in float64.

Sizes are generic: powers of two and odd numbers around them for tokens, widths and vocabularies.  Tokens are drawn
log-uniformly (a vocabulary sorted by frequency: a few tokens make up most of a text), gates around sigmoid(2).
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decoding step of a batch: 16 tokens looked up, where the call itself is what counts
        {"name": "lookup step", "op": "lookup", "n": 16, "vocab": 32000, "width": 2048, "dtype": "bf16"},
        # the lookup of a large training batch
        {"name": "lookup batch", "op": "lookup", "n": 65536, "vocab": 131072, "width": 4096, "dtype": "bf16"},
        # gradient of a micro-batch of 8 sequences of 2048 tokens
        {"name": "embedding gradient", "op": "lookup_grad", "n": 16384, "vocab": 32000, "width": 2048, "dtype": "bf16", "pad": 0.05},
        # gradient of a large batch and vocabulary
        {"name": "embedding gradient large", "op": "lookup_grad", "n": 65536, "vocab": 131072, "width": 4096, "dtype": "bf16", "pad": 0.0},
        # odd sizes in float32, a fifth of the batch is padding
        {"name": "embedding gradient odd", "op": "lookup_grad", "n": 5003, "vocab": 50257, "width": 769, "dtype": "f32", "pad": 0.2},
        # one decoding step of 32 requests: the state moves on by one token
        {"name": "scan step", "op": "scan", "batch": 32, "length": 1, "width": 2048, "dtype": "bf16", "ragged": False, "grad": False},
        # a training step's forward and backward pass
        {"name": "scan training", "op": "scan", "batch": 8, "length": 2048, "width": 2048, "dtype": "bf16", "ragged": False, "grad": True},
        # prefill of one very long sequence
        {"name": "scan long", "op": "scan", "batch": 1, "length": 65536, "width": 1024, "dtype": "bf16", "ragged": False, "grad": False},
        # packed sequences of uneven lengths, some empty, float32, forward and backward
        {"name": "scan ragged", "op": "scan", "batch": 37, "length": 1500, "width": 648, "dtype": "f32", "ragged": True, "grad": True},
        # sampling: a few rows, the chosen tokens' log probabilities and 20 alternatives
        {"name": "logprobs step", "op": "logprobs", "n": 8, "vocab": 131072, "dtype": "bf16", "top": 20, "masked": 0.0, "grad": False},
        # a policy-gradient or distillation step: log probabilities and entropies of 4096 tokens, and the gradient
        {"name": "logprobs training", "op": "logprobs", "n": 4096, "vocab": 131072, "dtype": "bf16", "top": 0, "masked": 0.0, "grad": True},
        # scoring a text in float32 with an odd vocabulary, part of which is masked, with 5 alternatives
        {"name": "logprobs odd", "op": "logprobs", "n": 1021, "vocab": 50257, "dtype": "f32", "top": 5, "masked": 0.1, "grad": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "lookup_grad", "scan", "scan", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    grain = rng.choice([1, 8, 64])                       # odd widths, and such as rows of 16 bytes allow
    if op in ("lookup", "lookup_grad"):
        width = max(1, _log(rng, 64, 4096) // grain) * grain
        vocab = _log(rng, 500, 131072)
        n = min(_log(rng, 1, 65536), (1 << 27) // width)
        case = {"op": op, "n": n, "vocab": vocab, "width": width, "dtype": dtype}
        if op == "lookup_grad":
            case["pad"] = rng.choice([0.0, 0.0, 0.1, 0.4])
        return case
    if op == "scan":
        width = max(1, _log(rng, 64, 4096) // grain) * grain
        length = rng.choice([1, _log(rng, 2, 65536), _log(rng, 2, 65536)])
        batch = _log(rng, 1, max(1, min(256, (1 << 25) // (width * length))))
        return {"op": op, "batch": batch, "length": length, "width": width, "dtype": dtype,
                "ragged": rng.random() < 0.4, "grad": rng.random() < 0.5}
    vocab = max(1, _log(rng, 1000, 131072) // grain) * grain
    n = min(_log(rng, 1, 8192), (1 << 28) // vocab)
    grad = rng.random() < 0.5
    return {"op": op, "n": n, "vocab": vocab, "dtype": dtype, "top": rng.choice([0, 1, 5, 20, 32]),
            "masked": rng.choice([0.0, 0.0, 0.3]), "grad": grad}


# --------------------------------------------------------------------------------------------------- the inputs

_SCALE = 0.75
_TEMPERATURE = 0.8


def _tokens(g, n, vocab):
    return (torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(vocab + 1.0)).long() - 1).clamp(0, vocab - 1)


def _lengths(case):
    """Lengths of a packed batch: uneven around the mean, some sequences empty; the total is batch * length."""
    b, total = case["batch"], case["batch"] * case["length"]
    r = np.random.RandomState(b * 1009 + case["length"])
    w = r.exponential(size=b) * (r.random_sample(b) > 0.1) + 1e-9
    n = np.floor(w / w.sum() * total).astype(np.int64)
    n[int(np.argmax(w))] += total - int(n.sum())
    return n


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, t = case["op"], _DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.empty(*shape, device="cuda", dtype=t).normal_(mean, std, generator=g)

    s = {"case": case}
    if op in ("lookup", "lookup_grad"):
        n, vocab, width = case["n"], case["vocab"], case["width"]
        s["tokens"] = _tokens(g, n, vocab)
        if op == "lookup":
            s["weight"] = normal(vocab, width)
        else:
            pad = torch.rand(n, generator=g, device="cuda") < case["pad"]
            s["tokens"] = torch.where(pad, -1, s["tokens"])
            s["grad"] = normal(n, width)
    elif op == "scan":
        b, length, width = case["batch"], case["length"], case["width"]
        shape = (b * length, width) if case["ragged"] else (b, length, width)
        s["x"], s["gate"] = normal(*shape), normal(*shape, mean=2.0, std=1.5)
        s["initial"] = torch.empty(b, width, device="cuda").normal_(generator=g)
        s["offsets"] = None
        if case["ragged"]:
            s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(_lengths(case))]).astype(np.int32)).cuda()
        if case["grad"]:
            s["grad"] = normal(*shape)
            s["grad_last"] = torch.empty(b, width, device="cuda").normal_(generator=g)
    else:
        n, vocab = case["n"], case["vocab"]
        s["logits"] = normal(n, vocab, std=3.0)
        s["tokens"] = torch.randint(0, vocab, (n,), generator=g, device="cuda")
        s["logits"][torch.arange(n, device="cuda"), s["tokens"]] += 8.0          # mostly likely tokens
        if case["masked"]:
            keep = torch.rand(vocab, generator=g, device="cuda") >= case["masked"]
            keep[0] = True
            s["logits"].masked_fill_(~keep, -math.inf)
            s["tokens"] = torch.where(keep[s["tokens"]], s["tokens"], 0)
        if case["grad"]:
            s["grad_logprobs"] = torch.empty(n, device="cuda").normal_(generator=g)
            s["grad_entropy"] = torch.empty(n, device="cuda").normal_(std=0.01, generator=g)
    return s


# ----------------------------------------------------------------------------------------------- the plain forms

def _plain_lookup(s):
    weight, tokens = s["weight"], s["tokens"]
    known = (tokens >= 0) & (tokens < weight.shape[0])
    rows = weight[torch.where(known, tokens, 0)].float() * _SCALE
    return torch.where(known[:, None], rows, 0.0).to(weight.dtype)


def _plain_lookup_grad(s):
    grad, tokens, vocab = s["grad"], s["tokens"], s["case"]["vocab"]
    known = (tokens >= 0) & (tokens < vocab)
    g = torch.where(known[:, None], grad.float() * _SCALE, 0.0)
    total = torch.zeros(vocab, grad.shape[1], device=grad.device)
    return total.index_add_(0, torch.where(known, tokens, 0), g).to(grad.dtype)


def _affine_scan(a, b, step, reverse):
    """h_t = a_t * h_{t-1} + b_t along dimension 1, by doubling: after the step of width w, (a, b) map the state
    2w tokens back to the state here."""
    if step >= a.shape[1]:
        return b
    if reverse:
        nb = torch.cat([b[:, :-step] + a[:, :-step] * b[:, step:], b[:, -step:]], 1)
        na = torch.cat([a[:, :-step] * a[:, step:], a[:, -step:]], 1)
    else:
        nb = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        na = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
    return _affine_scan(na, nb, 2 * step, reverse)


def _plain_scan(s):
    case, x, gate, initial, offsets = s["case"], s["x"], s["gate"], s["initial"], s["offsets"]
    width, dtype = x.shape[-1], x.dtype
    if offsets is None:                                   # a dense batch: its first and last rows
        b, length = x.shape[0], x.shape[1]
        first = torch.zeros(b, dtype=torch.long, device=x.device)
        last = torch.full((b,), length - 1, dtype=torch.long, device=x.device)
        where = (torch.arange(b, device=x.device), first), (torch.arange(b, device=x.device), last)
        some = torch.ones(b, dtype=torch.bool, device=x.device)
    else:                                                 # packed: one sequence of which some rows start anew
        b = offsets.shape[0] - 1
        lo, hi = offsets[:-1].long(), offsets[1:].long()
        some = hi > lo
        zero = torch.zeros_like(lo)
        where = (zero[some], lo[some]), (zero[some], hi[some] - 1)
        x, gate = x[None], gate[None]
    x32 = x.float()
    f, i = torch.sigmoid(gate.float()), torch.sigmoid(-gate.float())
    a, u = f.clone(), i * x32
    u[where[0]] += f[where[0]] * initial[some]
    a[where[0]] = 0.0                                     # the state before a sequence is in u already
    h = _affine_scan(a, u, 1, False)
    final = initial.clone()
    final[some] = h[where[1]]
    out = h.to(dtype)
    shape = s["x"].shape
    if not case["grad"]:
        return out.view(shape), final
    grad = s["grad"].view(x.shape).float()
    a, u = f.clone(), f * grad                            # what a token hands to the one before it
    u[where[1]] += f[where[1]] * s["grad_last"][some]
    a[where[1]] = 0.0
    mu = _affine_scan(a, u, 1, True)
    lam = grad.clone()
    lam[:, :-1] += mu[:, 1:]
    if offsets is not None:                               # nothing is handed from one sequence to another
        lam[where[1]] = grad[where[1]]
    lam[where[1]] += s["grad_last"][some]
    before = torch.empty_like(h)
    before[:, 1:] = h[:, :-1]
    before[where[0]] = initial[some]
    dx = (i * lam).to(dtype)
    dgate = (lam * (before - x32) * f * i).to(dtype)
    dinitial = s["grad_last"].clone()
    dinitial[some] = mu[where[0]]
    return out.view(shape), final, dx.view(shape), dgate.view(shape), dinitial


def _plain_logprobs(s):
    case, logits, tokens = s["case"], s["logits"], s["tokens"]
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    d = (x - top) / _TEMPERATURE
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    logsum = torch.log(total)
    empty = total == 0.0
    logp = torch.where(empty, -math.inf, d - logsum)
    p = torch.where(empty, 0.0, e / total)
    plogp = torch.where(p > 0.0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    known = (tokens >= 0) & (tokens < x.shape[1])
    at = torch.where(known, tokens, 0)[:, None]
    out = [torch.where(known, logp.gather(1, at)[:, 0], 0.0), entropy]
    if case["top"]:
        # one key for each value that orders by value, then by index, lowest first
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) - torch.arange(x.shape[1], device=x.device)
        index = torch.topk(key, case["top"], dim=1).indices
        out += [logp.gather(1, index), index]
    if case["grad"]:
        g, ge = s["grad_logprobs"][:, None], s["grad_entropy"][:, None]
        one = torch.zeros_like(x).scatter_(1, at, known[:, None].float())
        dx = torch.where(known[:, None], g, 0.0) * (one - p) - ge * (plogp + p * entropy[:, None])
        dx = torch.where(empty, 0.0, dx)                  # a row whose mask leaves nothing has no gradient
        out.append((dx / _TEMPERATURE).to(logits.dtype))
    return out


# ------------------------------------------------------------------------------------------------------- one pass

def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        return {"lookup": _plain_lookup, "lookup_grad": _plain_lookup_grad, "scan": _plain_scan, "logprobs": _plain_logprobs}[op](state)
    import appy_b200 as appy
    if op == "lookup":
        return appy.embedding(state["weight"], state["tokens"], scale=_SCALE)
    if op == "lookup_grad":
        return appy.embedding_grad(state["grad"], state["tokens"], case["vocab"], scale=_SCALE)
    if op == "scan":
        x, gate, initial, offsets = state["x"], state["gate"], state["initial"], state["offsets"]
        h, last = appy.gated_scan(x, gate, initial, offsets)
        if not case["grad"]:
            return h, last
        return (h, last) + tuple(appy.gated_scan_grad(state["grad"], x, gate, h, initial, offsets, state["grad_last"]))
    r = appy.token_logprobs(state["logits"], state["tokens"], top=case["top"], temperature=_TEMPERATURE)
    out = [r.logprobs, r.entropy]
    if case["top"]:
        out += [r.top_logprobs, r.top_tokens]
    if case["grad"]:
        out.append(appy.token_logprobs_grad(state["logits"], state["tokens"], r.stats, state["grad_logprobs"], state["grad_entropy"],
                                            temperature=_TEMPERATURE))
    return out


# ---------------------------------------------------------------------------------------- what a pass cannot do without

def _distinct(n, vocab):
    """Expected number of different tokens among n drawn by _tokens."""
    edges = np.log(np.arange(1, vocab + 2, dtype=np.float64)) / math.log(vocab + 1.0)
    return float(np.sum(-np.expm1(n * np.log1p(-np.minimum(np.diff(edges), 1 - 1e-12)))))


def work(case):
    op, size = case["op"], _SIZES[case["dtype"]]
    if op == "lookup":
        n, width = case["n"], case["width"]
        return {"bytes": 8 * n + _distinct(n, case["vocab"]) * width * size + n * width * size, "flops": n * width}
    if op == "lookup_grad":
        n, width = case["n"], case["width"]
        live = n * (1 - case["pad"])
        return {"bytes": 8 * n + live * width * size + case["vocab"] * width * size, "flops": 2 * live * width}
    if op == "scan":
        elements, states = case["batch"] * case["length"] * case["width"], case["batch"] * case["width"] * 4
        w = {"bytes": 3 * elements * size + 2 * states, "flops": 10 * elements}
        if case["grad"]:                                  # gate, x, h and the gradient in, two gradients out
            w = {"bytes": w["bytes"] + 6 * elements * size + 3 * states, "flops": w["flops"] + 20 * elements}
        return w
    elements = case["n"] * case["vocab"]
    w = {"bytes": elements * size + case["n"] * (8 + 8 + case["top"] * 12), "flops": 6 * elements}
    if case["grad"]:
        w = {"bytes": w["bytes"] + 2 * elements * size + 16 * case["n"], "flops": w["flops"] + 10 * elements}
    return w


# -------------------------------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"lookup": _exact_lookup, "lookup_grad": _exact_lookup_grad, "scan": _exact_scan, "logprobs": _exact_logprobs}[case["op"]](case, s)


def _exact_lookup(case, s):
    return torch.nn.functional.embedding(s["tokens"], s["weight"]).double() * _SCALE


def _exact_lookup_grad(case, s):
    order = torch.argsort(s["tokens"], stable=True)
    order = order[int((s["tokens"] < 0).sum()):]
    out = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
    for part in torch.split(order, 4096):
        out.index_put_((s["tokens"][part],), s["grad"][part].double() * _SCALE, accumulate=True)
    return out


def _exact_scan(case, s):
    b, length, width = case["batch"], case["length"], case["width"]
    if case["ragged"]:
        lens = _lengths(case)
        longest = int(lens.max())
        if longest > 70000:
            return None
        lo = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)])[:-1]).cuda()
        n = torch.from_numpy(lens).cuda()
    else:
        longest = length
        lo, n = torch.arange(b, device="cuda") * length, torch.full((b,), length, device="cuda")
    rows = case["batch"] * case["length"]
    x, gate = s["x"].view(rows, width), s["gate"].view(rows, width)
    h = s["initial"].double()
    out = torch.empty(rows, width, dtype=torch.float64, device="cuda")
    for t in range(longest):
        on = (n > t).nonzero()[:, 0] if case["ragged"] else slice(None)
        at = lo[on] + t
        f = torch.sigmoid(gate[at].double())
        h[on] = f * h[on] + (1 - f) * x[at].double()
        out[at] = h[on]
    shape = s["x"].shape
    if not case["grad"]:
        return out.view(shape), h
    lam = s["grad_last"].double()
    dx, dgate = torch.empty_like(out), torch.empty_like(out)
    for t in reversed(range(longest)):
        on = (n > t).nonzero()[:, 0] if case["ragged"] else slice(None)
        at = lo[on] + t
        f = torch.sigmoid(gate[at].double())
        before = s["initial"].double()[on] if t == 0 else out[at - 1]
        total = lam[on] + s["grad"].view(rows, width)[at].double()
        dx[at] = total * (1 - f)
        dgate[at] = total * (before - x[at].double()) * f * (1 - f)
        lam[on] = total * f
    return out.view(shape), h, dx.view(shape), dgate.view(shape), lam


def _exact_logprobs(case, s):
    parts = []
    for rows in torch.split(torch.arange(case["n"], device="cuda"), max(1, (1 << 25) // case["vocab"])):
        z = s["logits"][rows].double()
        logp = torch.log_softmax(z / _TEMPERATURE, -1)
        p = logp.exp()
        entropy = torch.special.entr(p).sum(-1)
        got = [logp[torch.arange(len(rows), device="cuda"), s["tokens"][rows]], entropy]
        if case["top"]:
            got.append(logp.sort(dim=-1, descending=True).values[:, :case["top"]])
        if case["grad"]:
            g, ge = s["grad_logprobs"][rows].double()[:, None], s["grad_entropy"][rows].double()[:, None]
            dz = -g * p - ge * (p * logp.clamp_min(-1e300) + p * entropy[:, None])
            dz[torch.arange(len(rows), device="cuda"), s["tokens"][rows]] += g[:, 0]
            got.append((dz / _TEMPERATURE))
        parts.append(got)
    out = [torch.cat(c) for c in zip(*parts)]
    return out[:3] + [None] + out[3:] if case["top"] else out
