"""The operators of on-policy distillation: a student writes its own continuations and is taught on what it wrote.

* `head`     hidden states to logits through a head held in 8 bits (`quantize_blocks`, `matmul_blocks`): one scale for every 128
             values of a hidden state, one for every 128 x 128 weights;
* `sample`   logits to tokens (`sample_rows`): temperature, top-k, top-p and min-p, from given random numbers;
* `lookup`   tokens to hidden states (`embed_rows`), and `grad`, the embedding's gradient (`embed_grad`);
* `rest`     the loss on what was written (`div_topk_rest`): the generalised Jensen-Shannon divergence between the stored top
             entries of a teacher with the rest of its vocabulary as one more outcome and the student's, with its gradient.

`run` computes each in torch operations in 32 bits (`own` false), or through the framework's own calls (`own` true).
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
REST_MIN = 2.0 ** -14


def listed():
    return [
        # one token for one conversation, a 32k vocabulary, usual settings
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "pitch": 32000, "dtype": "bf16", "set": "usual", "banned": 0.0},
        # a step of a large batch of rollouts, a 128k vocabulary, every row with settings of its own
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 128256, "pitch": 128256, "dtype": "bf16", "set": "mixed", "banned": 0.01},
        # many candidates at once from fp32 logits of an odd vocabulary: whole prompts' rows, plain temperature sampling and nuclei
        {"name": "sample_many", "op": "sample", "rows": 2048, "vocab": 50257, "pitch": 50257, "dtype": "fp32", "set": "wide", "banned": 0.0},
        # the tokens of a full training batch, a scaled embedding
        {"name": "lookup_batch", "op": "lookup", "tokens": 32768, "vocab": 128256, "width": 4096, "dtype": "bf16", "itype": "int64", "padding": 0.1},
        # the gradient of one short exchange, added to what a tied head has left in the gradient
        {"name": "grad_short", "op": "grad", "tokens": 131, "vocab": 32000, "width": 1024, "dtype": "fp32", "itype": "int64", "padding": 0.0, "into": True},
        # the gradient of a full training batch, a whole new one
        {"name": "grad_batch", "op": "grad", "tokens": 32768, "vocab": 128256, "width": 2048, "dtype": "bf16", "itype": "int64", "padding": 0.1, "into": False},
        # the loss on one short exchange, fp32 logits
        {"name": "rest_short", "op": "rest", "rows": 131, "vocab": 32000, "pitch": 32000, "k": 400, "beta": 0.5, "T": 1.0, "dtype": "fp32", "masked": 0.0},
        # forward KL with the rest, an odd vocabulary without padding, odd row count, padding tokens among the rows
        {"name": "rest_50257_odd", "op": "rest", "rows": 4093, "vocab": 50257, "pitch": 50257, "k": 100, "beta": 0.0, "T": 1.5, "dtype": "bf16", "masked": 0.1},
        # the loss on a large batch of a 128k vocabulary
        {"name": "rest_128k", "op": "rest", "rows": 8192, "vocab": 128256, "pitch": 128256, "k": 200, "beta": 0.5, "T": 1.0, "dtype": "bf16", "masked": 0.0},
        # the head for one token: the weights have to be read
        {"name": "head_one", "op": "head", "rows": 1, "vocab": 128256, "width": 4096, "dtype": "bf16"},
        # the head for a batch of rollouts on an odd vocabulary
        {"name": "head_rollouts", "op": "head", "rows": 61, "vocab": 50257, "width": 2048, "dtype": "bf16"},
        # the head for whole conversations: a matrix product
        {"name": "head_batch", "op": "head", "rows": 8192, "vocab": 128256, "width": 4096, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _vocab(rng, most=200064):
    """A vocabulary a tokenizer has, or any width."""
    if rng.random() < 0.5:
        return rng.choice([v for v in (32000, 32100, 50257, 50304, 100277, 128256, 151665, 151936) if v <= most])
    return _log(rng, 4000, most)


def _pitch(rng, vocab):
    """Columns of the stored rows: the vocabulary's own, or padded as model heads are."""
    return rng.choice([vocab, -(-vocab // 64) * 64, -(-vocab // 256) * 256])


def draw(rng):
    op = rng.choice(["sample", "sample", "lookup", "grad", "rest", "rest", "head", "head"])
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "sample":
        v = _vocab(rng)
        return {"op": op, "rows": max(1, min(_log(rng, 1, 4096), 100_000_000 // v)), "vocab": v, "pitch": _pitch(rng, v), "dtype": dt,
                "set": rng.choice(["usual", "mixed", "wide", "plain"]), "banned": rng.choice([0.0, 0.01, 0.5])}
    if op in ("lookup", "grad"):
        v, w = _vocab(rng), rng.choice([1024, 2048, 4096, 8 * rng.randrange(33, 600, 2), rng.randrange(257, 4800, 2)])
        if op == "grad":
            v = min(v, 4 * 128256 * 2048 // (2 * BYTES[dt] * w))
        c = {"op": op, "tokens": min(_log(rng, 1, 65536), 134_000_000 // w), "vocab": v, "width": w, "dtype": dt,
             "itype": rng.choice(["int64", "int32"]), "padding": rng.choice([0.0, 0.1, 0.4])}
        return {**c, "into": rng.random() < 0.4} if op == "grad" else c
    if op == "rest":
        v = _vocab(rng)
        return {"op": op, "rows": max(1, min(_log(rng, 1, 16384), 4 * 8192 * 128256 // (2 * BYTES[dt] * v))), "vocab": v, "pitch": _pitch(rng, v),
                "k": _log(rng, 10, 500), "beta": rng.choice([0.0, 0.1, 0.5, 0.9, 1.0]), "T": rng.choice([1.0, 1.5, 2.0]), "dtype": dt,
                "masked": rng.choice([0.0, 0.1, 0.3])}
    v, w = _vocab(rng), rng.choice([1024, 2048, 4096, 128 * rng.randrange(5, 40, 2), rng.randrange(501, 5000, 2)])
    return {"op": op, "rows": max(1, min(_log(rng, 1, 8192), int(8192 * 128256 * 4096 / (v * w)))), "vocab": v, "width": w, "dtype": rng.choice(["bf16", "bf16", "fp16"])}


# ------------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(n, m, dtype, g, std=1.0):
    x = torch.empty((n, m), dtype=dtype, device=DEV)
    for a in range(0, n, 4096):
        b = min(n, a + 4096)
        x[a:b] = torch.randn((b - a, m), generator=g, device=DEV, dtype=dtype) * std
    return x


def _tokens(n, vocab, itype, padding, g):
    """Token ids as text has them: a few ids make up most of it; padding tokens are negative."""
    r = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    t = (r.pow(4) * vocab).long().clamp_(max=vocab - 1)
    t = torch.where(torch.rand(n, generator=g, device=DEV) < padding, torch.full_like(t, -1), t)
    return t.to(getattr(torch, itype))


def _stored_rows(n, vocab, k, g):
    """Top-K rows as the dataset holds them: distinct ids, crowded towards the low ids, fp16 log-probs that hold most of the mass."""
    edge = torch.linspace(0, 1, k + 1, device=DEV, dtype=torch.float64).square().mul(vocab - k).long() + torch.arange(k + 1, device=DEV)
    low, width = edge[:-1], edge[1:] - edge[:-1]
    ids = low + (torch.rand((n, k), generator=g, device=DEV) * width).long().clamp_(max=width - 1)
    ids = torch.gather(ids, 1, torch.rand((n, k), generator=g, device=DEV).argsort(1))
    score = torch.randn((n, k), generator=g, device=DEV) * 2.5
    rest = torch.rand((n, 1), generator=g, device=DEV) * 0.2 + 0.005
    logp = torch.log_softmax(score.sort(1, descending=True).values, 1) + torch.log1p(-rest)
    return logp.half(), ids.to(torch.int32)


def _settings(kind, rows, g):
    """Per-row (temperature, top_k, top_p, min_p)."""
    one = torch.ones(rows, device=DEV)
    pick = lambda v: torch.tensor(v, device=DEV)[torch.randint(len(v), (rows,), generator=g, device=DEV)]  # noqa: E731
    if kind == "plain":                              # the student's own distribution
        return one, torch.zeros(rows, dtype=torch.int32, device=DEV), one, torch.zeros(rows, device=DEV)
    if kind == "usual":
        return one * 0.8, torch.full((rows,), 50, dtype=torch.int32, device=DEV), one * 0.95, one * 0.05
    if kind == "wide":                               # large nuclei and none
        return pick([1.0, 1.0, 1.3]), torch.zeros(rows, dtype=torch.int32, device=DEV), pick([1.0, 0.98, 0.9]), torch.zeros(rows, device=DEV)
    return pick([0.0, 0.6, 0.8, 1.0, 1.5]), pick([0, 0, 1, 20, 50, 400]).int(), pick([1.0, 0.98, 0.9, 0.5]), pick([0.0, 0.0, 0.02, 0.1])


def _prepare_sample(c, g):
    n, v, p = c["rows"], c["vocab"], c["pitch"]
    x = _normal(n, p, DTYPES[c["dtype"]], g, 2.0)
    k = min(64, v)                                   # what the text makes likely stands out, the first of it the most
    at = torch.randint(v, (n, k), generator=g, device=DEV)
    x.scatter_(1, at, (14.0 - torch.arange(k, device=DEV) * 0.12 + torch.randn((n, k), generator=g, device=DEV) * 1.5).to(x.dtype))
    if c["banned"]:
        x.masked_fill_((torch.rand((1, p), generator=g, device=DEV) < c["banned"]), float("-inf"))
    s = _settings(c["set"], n, g)
    return {"x": x[:, :v], "u": torch.rand(n, generator=g, device=DEV), "T": s[0], "top_k": s[1], "top_p": s[2], "min_p": s[3]}


def _prepare_rest(c, g):
    n, v, k = c["rows"], c["vocab"], c["k"]
    masked = torch.rand(n, generator=g, device=DEV) < c["masked"]
    row_map = torch.where(masked, -1, (~masked).long().cumsum(0) - 1).int()
    val, idx = _stored_rows(n, v, k, g)
    x = _normal(n, c["pitch"], DTYPES[c["dtype"]], g, 2.0)
    near = val[row_map.clamp_min(0).long()].float() + math.log(v) + 4.0 + torch.randn((n, k), generator=g, device=DEV)
    x.scatter_(1, idx[row_map.clamp_min(0).long()].long(), (near * c["T"]).to(x.dtype))
    return {"x": x[:, :v], "val": val, "idx": idx, "row_map": row_map, "scale": 1.0 / n}


def _blocks(v):
    return -(-v // 128)


def _prepare_head(c, g):
    """The hidden states, and the head's weights as they are kept: 8-bit values [vocab, whole blocks of columns] with zeros behind
    the last column, and a scale for every 128 x 128 of them."""
    v, w = c["vocab"], c["width"]
    codes = torch.zeros((v, _blocks(w) * 128), dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.empty((_blocks(v), _blocks(w)), device=DEV)
    for a in range(0, v, 16384):
        b = min(v, a + 16384)
        part = torch.zeros((_blocks(b - a) * 128, _blocks(w) * 128), device=DEV)
        part[: b - a, :w] = torch.randn((b - a, w), generator=g, device=DEV) * 0.02 * (1 + torch.rand((b - a, 1), generator=g, device=DEV))
        part = part.view(_blocks(b - a), 128, _blocks(w), 128)
        s = part.abs().amax((1, 3)) / 448.0
        scales[a // 128:a // 128 + _blocks(b - a)] = s
        codes[a:b] = (part / s[:, None, :, None]).view(_blocks(b - a) * 128, -1)[: b - a].to(torch.float8_e4m3fn)
    h = _normal(c["rows"], w, DTYPES[c["dtype"]], g)
    h *= torch.exp(torch.randn((1, w), generator=g, device=DEV)).to(h.dtype)        # some channels are far larger than others
    return {"h": h, "codes": codes, "scales": scales}


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "sample":
        s = _prepare_sample(case, g)
    elif op == "rest":
        s = _prepare_rest(case, g)
    elif op == "head":
        s = _prepare_head(case, g)
    else:
        n, v, w, dt = case["tokens"], case["vocab"], case["width"], DTYPES[case["dtype"]]
        s = {"tokens": _tokens(n, v, case["itype"], case["padding"], g), "scale": math.sqrt(w)}
        if op == "lookup":
            s["table"] = _normal(v, w, dt, g, 0.02)
        else:
            s["grad"] = _normal(n, w, dt, g, 0.01)
            s["into"] = _normal(v, w, dt, g, 0.01) if case["into"] else None
    return {"case": case, **s}


# ------------------------------------------------------------------------------------------------ the plain forms

LOG2E = 1.4426950408889634
#: 2^f on [-1/2, 1/2], from the highest power down: products and sums are rounded one by one
EXP2 = (0.001326472731307149, 0.009671512991189957, 0.05550733581185341, 0.24022242426872253, 0.6931470036506653, 1.0)


def _share(mass, part):
    """floor(mass * part / 2^24) of whole numbers, `part` <= 2^24, without leaving 64 bits."""
    return (mass >> 24) * part + (((mass & 0xffffff) * part) >> 24)


def _plain_sample(s):
    """Weights are whole numbers of 2^-31 of the largest one's, so that every sum is exact and the token does not depend on any order.
    Tokens go in descending order of their logits, equal ones by their index."""
    x, T = s["x"].float(), s["T"].unsqueeze(1)
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    rate = torch.where(T > 0, torch.tensor(LOG2E, device=x.device) / T, math.inf)
    t = torch.where(x == top, 0.0, (x - top) * rate)
    t = torch.where(t >= -64.0, t, -64.0)                                            # NaN as well
    n = t.round()
    f = t - n
    p = torch.full_like(f, EXP2[0])
    for c in EXP2[1:]:
        p = p * f + c
    p = p * ((n.int() + 127) << 23).view(torch.float32)                              # times 2^n
    weight = (p * 2.0 ** 31).long()
    x, at = x.sort(dim=1, descending=True, stable=True)
    w = weight.gather(1, at)
    upto = w.cumsum(1)
    before = upto - w
    rank = torch.arange(x.shape[1], device=x.device).unsqueeze(0)
    k = torch.where(T[:, 0] > 0, s["top_k"].long(), 1).unsqueeze(1)
    keep = (w > 0) & ((k <= 0) | (rank < k))
    mass = torch.where(keep, w, 0).sum(1, keepdim=True)
    top_p = s["top_p"].unsqueeze(1)
    limit = _share(mass, (top_p.clamp(0, 1) * 2.0 ** 24).long()).clamp_min(1)
    keep &= ~(top_p < 1) | (before < limit)
    least = (s["min_p"].clamp(0, 1) * 2.0 ** 31).long().unsqueeze(1)
    keep &= (w < least).long().cumsum(1) == 0
    mass = torch.where(keep, w, 0).sum(1, keepdim=True)
    want = _share(mass, (s["u"].clamp(0, 1) * 2.0 ** 24).long().clamp_max(2 ** 24 - 1).unsqueeze(1))
    place = (upto <= want).long().sum(1, keepdim=True).clamp_max(x.shape[1] - 1)
    token = at.gather(1, place)
    logp = (t.gather(1, token) - p.sum(1, keepdim=True).log2()) * math.log(2.0)
    empty = torch.isneginf(top)
    token, logp = torch.where(empty, -1, token), torch.where(empty, -math.inf, logp)
    return {"tokens": token[:, 0], "logp": logp[:, 0], "kept": torch.where(empty, 0, keep.long().sum(1, keepdim=True))[:, 0].int()}


def _plain_lookup(s):
    table, t = s["table"], s["tokens"].long()
    inside = (t >= 0) & (t < table.shape[0])
    rows = table[torch.where(inside, t, 0)].float() * s["scale"]
    return {"hidden": torch.where(inside.unsqueeze(1), rows, 0.0).to(table.dtype)}


def _plain_grad(s):
    t, g, v = s["tokens"].long(), s["grad"].float(), s["case"]["vocab"]
    inside = (t >= 0) & (t < v)
    total = torch.zeros((v, g.shape[1]), device=g.device).index_add_(0, t[inside], g[inside]) * s["scale"]
    if s["into"] is None:
        return {"grad": total.to(s["grad"].dtype)}
    return {"grad": s["into"].copy_((s["into"].float() + total))}


def _plain_rest(s):
    c, x = s["case"], s["x"]
    z = x.float() * (1.0 / c["T"])
    at = s["row_map"].clamp_min(0).long()
    live = (s["row_map"] >= 0).unsqueeze(1)
    ids, lp = s["idx"][at].long(), s["val"][at].float()
    beta = c["beta"]
    listed = torch.zeros(z.shape, dtype=torch.bool, device=z.device).scatter_(1, ids, True)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True).log() + top
    others = torch.where(listed, 0.0, e)
    left = others.sum(1, keepdim=True)
    lq = torch.cat([z.gather(1, ids) - total, left.log() + top - total], 1)          # the K entries and the rest
    p0 = (1.0 - lp.exp().sum(1, keepdim=True)).clamp_min(REST_MIN)
    lp = torch.cat([lp, p0.log()], 1)
    lp = lp - lp.exp().sum(1, keepdim=True).log()
    p, q, r = lp.exp(), lq.exp(), lp - lq
    if beta == 0.0:
        loss, slope = (p * r).sum(1), -p
    elif beta == 1.0:
        loss, slope = -(q * r).sum(1), -q * r
    else:
        above = torch.log1p(beta * torch.expm1(r))                                   # log of the mixture over the student
        loss = (beta * p * (r - above) - (1 - beta) * q * above).sum(1)
        slope = -(1 - beta) * q * above                                              # the probability times the derivative by it
    d = slope - q * slope.sum(1, keepdim=True)
    scale = s["scale"] / c["T"]
    grad = others / left * (d[:, -1:] * scale)
    grad = grad.scatter_(1, ids, d[:, :-1] * scale)
    return {"loss": torch.where(live[:, 0], loss, 0.0), "grad": torch.where(live, grad, 0.0).to(x.dtype)}


def _plain_head(s):
    h, codes, scales = s["h"].float(), s["codes"], s["scales"]
    n, w, wide = h.shape[0], h.shape[1], codes.shape[1]
    h = torch.nn.functional.pad(h, (0, wide - w)).view(n, wide // 128, 128)
    own_scale = (h.abs().amax(2, keepdim=True) / 448.0).clamp_min(2.0 ** -100)
    h = ((h / own_scale).to(torch.float8_e4m3fn).float() * own_scale).view(n, wide)
    full = scales.repeat_interleave(128, 0)[: codes.shape[0]].repeat_interleave(128, 1)
    return {"logits": (h @ (codes.float() * full).t()).to(s["h"].dtype)}


# ------------------------------------------------------------------------------------------------ the framework's calls

def _own(s):
    import llm_distillery_amd as D
    c = s["case"]
    op = c["op"]
    if op == "sample":
        tokens, logp, kept = D.sample_rows(s["x"], s["u"], temperature=s["T"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logp": logp, "kept": kept}
    if op == "lookup":
        return {"hidden": D.embed_rows(s["table"], s["tokens"], scale=s["scale"])}
    if op == "grad":
        return {"grad": D.embed_grad(s["grad"], s["tokens"], c["vocab"], scale=s["scale"], into=s["into"])}
    if op == "rest":
        loss, grad = D.div_topk_rest(c["beta"], s["x"], s["val"], s["idx"], row_map=s["row_map"], T=c["T"], rest_min=REST_MIN, grad_scale=s["scale"])
        return {"loss": loss, "grad": grad}
    head = D.BlockQuantized(s["codes"], s["scales"], c["width"])
    return {"logits": D.matmul_blocks(D.quantize_blocks(s["h"]), head, dtype=s["h"].dtype)}


def run(state):
    if own:
        return _own(state)
    return {"sample": _plain_sample, "lookup": _plain_lookup, "grad": _plain_grad, "rest": _plain_rest, "head": _plain_head}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def _exact_sample(c, s):
    if c["rows"] * c["vocab"] > 40_000_000:
        return None
    logits = s["x"].float().cpu().numpy()
    u, T, top_k, top_p, min_p = (s[k].cpu().numpy() for k in ("u", "T", "top_k", "top_p", "min_p"))
    logp = np.empty(c["rows"])
    one = np.float32
    for i, x in enumerate(logits):
        x = np.where(np.isnan(x), one(-np.inf), x)
        if x.max() == -np.inf:
            logp[i] = -np.inf
            continue
        likely = np.flatnonzero(x == x.max()) if T[i] <= 0 else np.flatnonzero((x - x.max()) * (one(LOG2E) / T[i]) > -33)
        likely = likely[np.argsort(-x[likely], kind="stable")]
        d = (x[likely] - x.max()) * (one(LOG2E) / T[i]) if T[i] > 0 else np.zeros(len(likely), one)
        whole = np.rint(d)
        f = d - whole
        p = np.full_like(f, one(EXP2[0]))
        for k in EXP2[1:]:
            p = p * f + one(k)
        w = np.floor(np.ldexp(p.astype(np.float64), whole.astype(np.int64) + 31)).astype(object)
        w = [int(v) for v in w if v > 0]
        k = 1 if T[i] <= 0 else int(top_k[i])
        w = w[:k] if k > 0 else w
        if top_p[i] < 1:
            limit = max(1, sum(w) * int(max(0.0, float(top_p[i])) * 2 ** 24) // 2 ** 24)
            end, mass = 0, 0
            while end < len(w) and mass < limit:
                mass, end = mass + w[end], end + 1
            w = w[:end]
        least = int(min(1.0, max(0.0, float(min_p[i]))) * 2 ** 31)
        end = next((j for j, v in enumerate(w) if v < least), len(w))
        w = w[:end]
        want = sum(w) * min(2 ** 24 - 1, int(float(u[i]) * 2 ** 24)) // 2 ** 24
        j, mass = 0, w[0]
        while mass <= want:
            j += 1
            mass += w[j]
        if T[i] <= 0:
            logp[i] = -math.log(len(likely))
        else:
            z = x.astype(np.float64) / float(T[i])
            logp[i] = z[likely[j]] - z.max() - math.log(np.exp(z - z.max()).sum())
    return {"tokens": None, "logp": logp, "kept": None}


def _exact_embedding(c, s):
    t = s["tokens"].long()
    inside = ((t >= 0) & (t < c["vocab"])).nonzero()[:, 0]
    if c["op"] == "lookup":
        out = torch.zeros((c["tokens"], c["width"]), dtype=torch.float64, device=DEV)
        out[inside] = s["table"].double()[t[inside]] * s["scale"]
        return {"hidden": out}
    out = torch.zeros((c["vocab"], c["width"]), dtype=torch.float64, device=DEV)
    out.index_add_(0, t[inside], s["grad"][inside].double())
    out *= s["scale"]
    return {"grad": out if s["into"] is None else out + s["into"].double()}


def _exact_rest(c, s):
    beta, v = c["beta"], c["vocab"]
    loss = torch.zeros(c["rows"], dtype=torch.float64, device=DEV)
    grad = torch.zeros((c["rows"], v), dtype=torch.float64, device=DEV)
    rows = (s["row_map"] >= 0).nonzero()[:, 0]
    for part in rows.split(512):
        at = s["row_map"][part].long()
        ids = s["idx"][at].long()
        q = torch.softmax(s["x"][part].double() / c["T"], 1)
        lq = torch.log_softmax(s["x"][part].double() / c["T"], 1)
        p = s["val"][at].double().exp()
        p = torch.cat([p, (1 - p.sum(1, keepdim=True)).clamp_min(REST_MIN)], 1)
        p = p / p.sum(1, keepdim=True)
        others = lq.scatter(1, ids, -math.inf)
        l0 = torch.logsumexp(others, 1, keepdim=True)
        lk = torch.cat([lq.gather(1, ids), l0], 1)
        k = lk.exp()
        if beta == 0.0:
            value, by_q = p * (p.log() - lk), -p / k
        elif beta == 1.0:
            value, by_q = k * (lk - p.log()), lk - p.log() + 1
        else:
            lm = (beta * p + (1 - beta) * k).log()
            value, by_q = beta * p * (p.log() - lm) + (1 - beta) * k * (lk - lm), (1 - beta) * (lk - lm)
        loss[part] = value.sum(1)
        mean = (k * by_q).sum(1, keepdim=True)
        g = q * (by_q[:, -1:] - mean)
        grad[part] = g.scatter(1, ids, k[:, :-1] * (by_q[:, :-1] - mean)) * (s["scale"] / c["T"])
    return {"loss": loss, "grad": grad}


def _exact_head(c, s):
    w, wide = c["width"], s["codes"].shape[1]
    h = torch.zeros((c["rows"], wide), device=DEV)
    h[:, :w] = s["h"].float()
    h = h.view(c["rows"], -1, 128)
    scale = torch.maximum(h.abs().amax(2) / 448.0, torch.tensor(2.0 ** -100, device=DEV))
    quotient = (h / scale.unsqueeze(2)).double()
    step = torch.exp2(torch.floor(torch.log2(quotient.abs().clamp_min(2.0 ** -9))).clamp_min(-6.0) - 3.0)
    h = (torch.round(quotient / step) * step * scale.double().unsqueeze(2)).view(c["rows"], wide)
    out = torch.empty((c["rows"], c["vocab"]), dtype=torch.float64, device=DEV)
    for a in range(0, c["vocab"], 16384):
        b = min(c["vocab"], a + 16384)
        block = torch.arange(a, b, device=DEV) // 128
        weights = (s["codes"][a:b].float().double().view(b - a, -1, 128) * s["scales"][block].double().unsqueeze(2)).view(b - a, wide)
        out[:, a:b] = h @ weights.t().contiguous()
    return {"logits": out}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    return _exact_sample(case, s) if op == "sample" else _exact_rest(case, s) if op == "rest" else _exact_head(case, s) if op == "head" \
        else _exact_embedding(case, s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

@functools.lru_cache(maxsize=None)
def _distinct(tokens, vocab, padding):
    """How many different ids _tokens() gives, as the mean over its draws."""
    edge = (torch.arange(vocab + 1, dtype=torch.float64) / vocab).pow(0.25)
    return float((1 - torch.pow(1 - (edge[1:] - edge[:-1]), tokens * (1 - padding))).sum())


def work(case):
    op = case["op"]
    if op == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * BYTES[case["dtype"]] + 5 * 4 + 8 + 4 + 4), "flops": case["rows"] * case["vocab"] * 4}
    if op == "rest":
        live = round(case["rows"] * (1 - case["masked"]))
        size = BYTES[case["dtype"]]
        return {"bytes": live * case["vocab"] * size + case["rows"] * case["vocab"] * size + live * case["k"] * 6 + case["rows"] * 8, "flops": live * case["vocab"] * 6}
    if op == "head":
        n, v, w = case["rows"], case["vocab"], case["width"]
        return {"bytes": v * _blocks(w) * 128 + _blocks(v) * _blocks(w) * 4 + n * w * BYTES[case["dtype"]] + n * v * BYTES[case["dtype"]], "flops": 2.0 * n * v * w}
    n, v, w, size = case["tokens"], case["vocab"], case["width"], BYTES[case["dtype"]]
    live, rows = n * (1 - case["padding"]), _distinct(n, v, case["padding"])
    if op == "lookup":
        return {"bytes": n * w * size + rows * w * size + n * 8, "flops": n * w}
    return {"bytes": live * w * size + n * 8 + (2 * rows * w * size if case["into"] else v * w * size), "flops": live * w}
