"""The operators at the ends of a token model and between its layers: what is measured of them.

``listed()`` and ``draw()`` give cases, ``prepare()`` the inputs a program holds before the call, ``run()`` one pass -
in elementary torch operations, or through ``cuv_b200`` where ``own`` is set - ``work()`` the bytes and operations a
pass cannot do without, ``exact()`` the same outputs in 64 bits.

Dense matrices are column-major, as everywhere in the package: a batch column (a token position) is contiguous.  Every
case is a dict with an ``op``:

``lookup``        dst[:, j] = scale * table[:, tok_j], a column of zeros where tok_j is padding (negative)
``lookup_grad``   dtable[:, v] = sum of dout[:, j] over the positions j with tok_j = v (the whole table is written)
``dropout``       dst = (u >= p ? src / (1 - p) : 0) [+ residual], u the generator's number of the element; the backward
                  pass is the same pass over the gradient
``logprob``       log probability of one given token per column, log-sum-exp, entropy, the ``top`` likeliest tokens
``logprob_grad``  gradient of those log probabilities (and of the entropies) with respect to the logits
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token for each of eight sequences being answered: latency of a single small call
        {"name": "lookup_step", "op": "lookup", "type": "bf16", "units": 4096, "vocab": 32768, "ncols": 8, "scale": 1.0,
         "pad": 0.0},
        # a training batch of 32768 token positions, embeddings scaled by sqrt(units)
        {"name": "lookup_batch", "op": "lookup", "type": "bf16", "units": 4096, "vocab": 65536, "ncols": 32768,
         "scale": 64.0, "pad": 0.0},
        # table gradient of a training batch: 16-bit activations' gradient, 32-bit table gradient
        {"name": "lookup_grad_batch", "op": "lookup_grad", "type": "bf16", "grad_type": "f32", "units": 4096,
         "vocab": 32768, "ncols": 16384, "pad": 0.0},
        # the same for odd sizes in 32 bits, a batch padded to its longest sequence
        {"name": "lookup_grad_odd", "op": "lookup_grad", "type": "f32", "grad_type": "f32", "units": 1023,
         "vocab": 50021, "ncols": 8191, "pad": 0.1},
        # dropout on the activations of a few columns: latency
        {"name": "dropout_small", "op": "dropout", "type": "f32", "units": 1024, "ncols": 64, "p": 0.5, "residual": False},
        # dropout of a layer's output added to the residual stream, a quarter of the units of the package's largest step
        {"name": "dropout_residual", "op": "dropout", "type": "bf16", "units": 16384, "ncols": 8192, "p": 0.1,
         "residual": True},
        # the backward pass over an odd matrix in half precision
        {"name": "dropout_odd", "op": "dropout", "type": "f16", "units": 4095, "ncols": 2049, "p": 0.25, "residual": False},
        # answering: four sequences, the sampled token's log probability and eight alternatives at a temperature of 0.7
        {"name": "logprob_step", "op": "logprob", "type": "bf16", "vocab": 131072, "ncols": 4, "scale": 1.4285714, "top": 8,
         "entropy": True, "masked": 0.0, "pad": 0.0},
        # training: log probabilities and entropies of a batch's target tokens
        {"name": "logprob_batch", "op": "logprob", "type": "bf16", "vocab": 32768, "ncols": 8192, "scale": 1.0, "top": 0,
         "entropy": True, "masked": 0.0, "pad": 0.0},
        # scoring prompts in 32 bits, an odd vocabulary, a third of it forbidden, twenty alternatives, padding
        {"name": "logprob_score", "op": "logprob", "type": "f32", "vocab": 50021, "ncols": 1000, "scale": 1.0, "top": 20,
         "entropy": True, "masked": 0.33, "pad": 0.05},
        # the training batch's gradient, with an entropy bonus in the loss
        {"name": "logprob_grad_batch", "op": "logprob_grad", "type": "bf16", "vocab": 32768, "ncols": 8192, "scale": 1.0,
         "entropy": True, "masked": 0.0, "pad": 0.0},
        # the gradient of a padded half-precision batch over an odd vocabulary
        {"name": "logprob_grad_odd", "op": "logprob_grad", "type": "f16", "vocab": 50021, "ncols": 777, "scale": 0.5,
         "entropy": False, "masked": 0.0, "pad": 0.2},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm, mostly odd and seldom round."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "dropout", "logprob", "logprob_grad"])
    kind = rng.choice(["f32", "f16", "bf16"])
    multiple = rng.choice([1, 1, 8, 64])         # half of the cases have no aligned columns

    def size(low, high):
        return max(low, _between(rng, low, high) // multiple * multiple)

    if op == "lookup":
        units, vocab = size(64, 8192), size(256, 131072)
        ncols = min(_between(rng, 1, 32768), 67_000_000 // units)
        return {"op": op, "type": kind, "units": units, "vocab": min(vocab, 400_000_000 // units), "ncols": ncols,
                "scale": rng.choice([1.0, math.sqrt(units)]), "pad": rng.choice([0.0, 0.1])}
    if op == "lookup_grad":
        units, vocab = size(64, 8192), size(256, 131072)
        ncols = min(_between(rng, 1, 65536), 67_000_000 // units)
        return {"op": op, "type": kind, "grad_type": rng.choice([kind, "f32"]), "units": units,
                "vocab": min(vocab, 90_000_000 // units), "ncols": ncols, "pad": rng.choice([0.0, 0.1])}
    if op == "dropout":
        units = size(64, 16384)
        return {"op": op, "type": kind, "units": units, "ncols": min(_between(rng, 1, 65536), 60_000_000 // units),
                "p": rng.choice([0.1, 0.25, 0.5]), "residual": rng.choice([True, False])}
    vocab = size(256, 131072)
    ncols = min(_between(rng, 1, 8192), 130_000_000 // vocab)
    case = {"op": op, "type": kind, "vocab": vocab, "ncols": ncols, "scale": rng.choice([1.0, 1.0, 1.25]),
            "entropy": rng.choice([True, False]), "masked": rng.choice([0.0, 0.0, 0.33]), "pad": rng.choice([0.0, 0.1])}
    if op == "logprob":
        case["top"] = rng.choice([0, 0, 1, 5, 20])
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------

def _columns(rows, cols, dtype):
    return torch.empty((cols, rows), dtype=dtype, device="cuda").t()


def _normal(g, rows, cols, dtype, spread=1.0):
    return (torch.randn((cols, rows), dtype=torch.float32, device="cuda", generator=g) * spread).to(dtype).t()


def _tokens(g, vocab, ncols, pad):
    """Token frequencies of text: rank r with a probability near 1/r; a share ``pad`` of the positions is padding (-1)."""
    u = torch.rand(ncols, dtype=torch.float64, device="cuda", generator=g)
    tok = ((u * math.log(vocab + 1.0)).exp().long() - 1).clamp_(0, vocab - 1)
    gone = torch.rand(ncols, device="cuda", generator=g) < pad
    return torch.where(gone, torch.full_like(tok, -1), tok)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, dtype = dict(case), TYPES[case["type"]]
    s = {"case": c}
    if c["op"] == "lookup":
        s["table"] = _normal(g, c["units"], c["vocab"], dtype, 0.02)
        s["tokens"] = _tokens(g, c["vocab"], c["ncols"], c["pad"])
        s["dst"] = _columns(c["units"], c["ncols"], dtype)
    elif c["op"] == "lookup_grad":
        s["dout"] = _normal(g, c["units"], c["ncols"], dtype)
        s["tokens"] = _tokens(g, c["vocab"], c["ncols"], c["pad"])
        s["dtable"] = _columns(c["units"], c["vocab"], TYPES[c["grad_type"]])
    elif c["op"] == "dropout":
        s["src"] = _normal(g, c["units"], c["ncols"], dtype)
        s["residual"] = _normal(g, c["units"], c["ncols"], dtype) if c["residual"] else None
        s["dst"] = _columns(c["units"], c["ncols"], dtype)
        s["seed"], s["step"], s["which"], s["col0"] = 0x9E3779B97F4A7C15 ^ seed, 17 + seed % 1000, 3, 5
    else:
        logits = _normal(g, c["vocab"], c["ncols"], dtype, 2.5)
        if c["masked"]:
            logits.masked_fill_((torch.rand(c["vocab"], device="cuda", generator=g) < c["masked"])[:, None], -math.inf)
        tok = torch.randint(0, c["vocab"], (c["ncols"],), device="cuda", generator=g)
        # a given token is one the column allows; of the few likeliest ones in half of the columns
        best = logits.argmax(0)
        likely = torch.rand(c["ncols"], device="cuda", generator=g) < 0.5
        allowed = torch.isfinite(logits.gather(0, tok[None])[0])
        tok = torch.where(likely | ~allowed, best, tok)
        gone = torch.rand(c["ncols"], device="cuda", generator=g) < c["pad"]
        s["logits"], s["tokens"] = logits, torch.where(gone, torch.full_like(tok, -1), tok)
        if c["op"] == "logprob_grad":
            z = logits.double() * float(np.float32(c["scale"]))
            lse = torch.logsumexp(z, 0)
            q = torch.exp(z - lse)
            s["lse"] = lse.float()
            s["entropy"] = (lse - (q * z.masked_fill(q == 0, 0.0)).sum(0)).float() if c["entropy"] else None
            s["dentropy"] = torch.full((c["ncols"],), 0.01 / c["ncols"], device="cuda") if c["entropy"] else None
            s["dlogp"] = torch.rand(c["ncols"], device="cuda", generator=g) - 1.0
            s["dlogits"] = _columns(c["vocab"], c["ncols"], dtype)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"lookup": _lookup, "lookup_grad": _lookup_grad, "dropout": _dropout, "logprob": _logprob,
            "logprob_grad": _logprob_grad}[s["case"]["op"]](s)


def _own(s):
    import cuv_b200 as cb
    c = s["case"]
    if c["op"] == "lookup":
        return cb.embedding(s["dst"], s["table"], s["tokens"], c["scale"])
    if c["op"] == "lookup_grad":
        return cb.embedding_grad(s["dtable"], s["tokens"], s["dout"])
    if c["op"] == "dropout":
        return cb.dropout(s["dst"], s["src"], c["p"], s["seed"], s["step"], s["col0"], s["which"], residual=s["residual"])
    if c["op"] == "logprob":
        r = cb.token_logprob(s["logits"], s["tokens"], scale=c["scale"], entropy=c["entropy"], top=c["top"])
        return {k: v for k, v in r._asdict().items() if v is not None}
    return cb.token_logprob_grad(s["dlogits"], s["logits"], s["lse"], s["tokens"], s["dlogp"], entropy=s["entropy"],
                                 dentropy=s["dentropy"], scale=c["scale"])


def _lookup(s):
    tok, table = s["tokens"], s["table"]
    picked = table.t()[tok.clamp(min=0)].float() * float(np.float32(s["case"]["scale"]))
    return torch.where((tok >= 0)[:, None], picked, 0.0).to(table.dtype).t()


def _lookup_grad(s):
    c, tok = s["case"], s["tokens"]
    rows = torch.zeros((c["vocab"], c["units"]), dtype=torch.float32, device="cuda")
    keep = (tok >= 0)[:, None]
    rows.index_add_(0, tok.clamp(min=0), torch.where(keep, s["dout"].t().float(), 0.0))
    return rows.to(TYPES[c["grad_type"]]).t()


_LOW = 0xFFFFFFFF


def _wide(a, b):
    """High and low word of the product of the 32-bit constant a and the 32-bit numbers b (held in 64 bits)."""
    return ((a >> 16) * b + (((a & 0xFFFF) * b) >> 16)) >> 16, (a * b) & _LOW


def _uniform(units, ncols, seed, step, which, col0):
    """The package's uniform numbers (Philox4x32-10): counter (row / 4, column, which, step), key = seed, one 32-bit word
    per row of four, its upper 24 bits as a number of [0, 1)."""
    groups = (units + 3) // 4
    x = torch.arange(groups, dtype=torch.int64, device="cuda")[None, :].expand(ncols, groups)
    y = (torch.arange(ncols, dtype=torch.int64, device="cuda") + col0)[:, None].expand(ncols, groups)
    z, w = torch.full_like(x, which), torch.full_like(x, step)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        (ph, pl), (qh, ql) = _wide(0xD2511F53, x), _wide(0xCD9E8D57, z)
        x, y, z, w = qh ^ y ^ k0, ql, ph ^ w ^ k1, pl
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([x, y, z, w], dim=2).reshape(ncols, 4 * groups)[:, :units]
    return (words >> 8).float() * 2.0 ** -24


def _dropout(s):
    c = s["case"]
    p = float(np.float32(c["p"]))
    u = _uniform(c["units"], c["ncols"], s["seed"], s["step"], s["which"], s["col0"])
    kept = torch.where(u >= p, s["src"].t().float() * float(np.float32(1.0 / (1.0 - p))), 0.0)
    if s["residual"] is not None:
        kept = kept + s["residual"].t().float()
    return kept.to(s["src"].dtype).t()


def _logprob(s):
    c, tok = s["case"], s["tokens"]
    scale = float(np.float32(c["scale"]))
    z = s["logits"].float() * scale
    m = z.amax(0)
    e = torch.exp(z - m)
    total = e.sum(0)
    lse = m + torch.log(total)
    out = {"lse": lse, "logp": torch.where(tok >= 0, z.gather(0, tok.clamp(min=0)[None])[0] - lse, 0.0)}
    if c["entropy"]:
        out["entropy"] = lse - (e * z.masked_fill(e == 0, 0.0)).sum(0) / total
    if c["top"]:
        value, index = torch.sort(s["logits"].t().float(), dim=1, descending=True, stable=True)
        value, index = value[:, :c["top"]] * scale - lse[:, None], index[:, :c["top"]]
        out["top_logp"] = value.t()
        out["top_index"] = torch.where(torch.isfinite(value), index, -1).int().t()
    return out


def _logprob_grad(s):
    c, tok = s["case"], s["tokens"]
    scale = float(np.float32(c["scale"]))
    logq = s["logits"].float() * scale - s["lse"]
    q = torch.exp(logq)
    dlogp = torch.where(tok >= 0, s["dlogp"], 0.0)
    d = -dlogp * q
    if c["entropy"]:
        d -= s["dentropy"] * q * (logq.masked_fill(q == 0, 0.0) + s["entropy"])
    d.scatter_add_(0, tok.clamp(min=0)[None], dlogp[None])
    return (d * scale).to(s["logits"].dtype)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _distinct(vocab, ncols, pad):
    """Expected number of distinct tokens among the positions (see _tokens)."""
    p = np.diff(np.log(np.arange(1, vocab + 2, dtype=np.float64))) / math.log(vocab + 1.0)
    return float(-np.expm1(ncols * (1.0 - pad) * np.log1p(-p)).sum())


def work(case):
    c, size = case, BYTES[case["type"]]
    if c["op"] == "lookup":
        n = c["units"] * c["ncols"]
        return {"bytes": int(n * size + _distinct(c["vocab"], c["ncols"], c["pad"]) * c["units"] * size + 8 * c["ncols"]),
                "flops": n}
    if c["op"] == "lookup_grad":
        n = int(c["units"] * c["ncols"] * (1.0 - c["pad"]))
        return {"bytes": n * size + 8 * c["ncols"] + c["units"] * c["vocab"] * BYTES[c["grad_type"]], "flops": n}
    if c["op"] == "dropout":
        n = c["units"] * c["ncols"]
        return {"bytes": n * size * (3 if c["residual"] else 2), "flops": n * (2 if c["residual"] else 1)}
    n = c["vocab"] * c["ncols"]
    if c["op"] == "logprob":
        return {"bytes": n * size + c["ncols"] * (16 + (4 if c["entropy"] else 0) + 8 * c["top"]),
                "flops": n * (6 if c["entropy"] else 4)}
    # a padded column's gradient is zero without an entropy term: it is written, its logits need not be read
    read = n if c["entropy"] else int(n * (1.0 - c["pad"]))
    return {"bytes": (read + n) * size + c["ncols"] * (16 + (8 if c["entropy"] else 0)), "flops": n * (8 if c["entropy"] else 5)}


# ---- the same outputs in 64 bits ---------------------------------------------------------------------------------

def _kept(c, s):
    """Which elements dropout keeps: the generator in unsigned 64-bit arithmetic, 256 columns at a time."""
    groups, low = (c["units"] + 3) // 4, np.uint64(_LOW)
    least = math.ceil(float(np.float32(c["p"])) * 2 ** 24)
    keep = np.empty((c["ncols"], c["units"]), dtype=bool)
    for first in range(0, c["ncols"], 256):
        n = min(256, c["ncols"] - first)
        ctr = np.zeros((4, n, groups), dtype=np.uint64)
        ctr[0] = np.arange(groups, dtype=np.uint64)
        ctr[1] = (np.arange(n, dtype=np.uint64) + np.uint64(first + s["col0"]))[:, None]
        ctr[2], ctr[3] = s["which"], s["step"]
        for r in range(10):
            k0 = np.uint64((s["seed"] + r * 0x9E3779B9) & _LOW)
            k1 = np.uint64(((s["seed"] >> 32) + r * 0xBB67AE85) & _LOW)
            a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            ctr = np.stack([(b >> np.uint64(32)) ^ ctr[1] ^ k0, b & low, (a >> np.uint64(32)) ^ ctr[3] ^ k1, a & low])
        keep[first:first + n] = ((ctr >> np.uint64(8)) >= least).transpose(1, 2, 0).reshape(n, 4 * groups)[:, :c["units"]]
    return keep


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "lookup":
        tok = s["tokens"].cpu()
        out = torch.zeros((c["ncols"], c["units"]), dtype=torch.float64)
        there = tok >= 0
        out[there] = s["table"].t().cpu()[tok[there]].double() * float(np.float32(c["scale"]))
        return out.t()
    if c["op"] == "lookup_grad":
        tok = s["tokens"].cpu().numpy()
        order = np.argsort(tok, kind="stable")
        order = order[tok[order] >= 0]
        out = np.zeros((c["vocab"], c["units"]))
        if order.size:
            values, starts = np.unique(tok[order], return_index=True)
            rows = s["dout"].t().cpu().double().numpy()[order]
            out[values] = np.add.reduceat(rows, starts, axis=0)
        return torch.from_numpy(out).t()
    if c["op"] == "dropout":
        keep = torch.from_numpy(_kept(c, s)).cuda()
        out = s["src"].t().double() / (1.0 - float(np.float32(c["p"]))) * keep
        return (out + s["residual"].t().double() if s["residual"] is not None else out).t()
    z = s["logits"].double() * float(np.float32(c["scale"]))
    tok = s["tokens"]
    if c["op"] == "logprob":
        logq = torch.log_softmax(z, 0)
        lse = torch.logsumexp(z, 0)
        out = {"lse": lse, "logp": torch.where(tok >= 0, logq.gather(0, tok.clamp(min=0)[None])[0], 0.0)}
        if c["entropy"]:
            out["entropy"] = torch.special.entr(logq.exp()).sum(0)
        if c["top"]:
            out["top_logp"] = torch.topk(logq, min(c["top"], c["vocab"]), dim=0).values
            out["top_index"] = None
        return out
    # the formula's log-sum-exp and entropy are inputs here, given in 32 bits
    q = torch.exp(z - s["lse"].double())
    weight = torch.where(tok >= 0, s["dlogp"].double(), 0.0)
    hot = torch.zeros_like(q)
    hot[tok.clamp(min=0), torch.arange(c["ncols"], device="cuda")] = 1.0
    out = weight * (hot - q)
    if c["entropy"]:
        out -= s["dentropy"].double() * (q * s["entropy"].double() - torch.special.entr(q))
    return out * float(np.float32(c["scale"]))
