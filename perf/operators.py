"""The operators around the sampler that a beam search over an 8-bit LM head runs, and what they are measured on.

  quantise   dlk_quantize_rows: 8-bit values and a scale for each row (hidden states: a token; weights: a channel)
  logits     dlk_logits_i8: the LM head's product in 8-bit integers, scales for each token and channel, soft-cap
  select     dlk_beam_select: the best continuations of each group of beams over the vocabulary
  reorder    dlk_beam_reorder: the beams' caches, small states and histories follow their parents

With `own` false `run` computes them in elementary torch operations, with `own` true through diskllm_amd.api.
"""
import math

import torch

own = False

GRAMMAR_ROW = 36          # bytes of a dlk_grammar_row: a beam's grammar position


def _quantise(name, rows, n, dtype, pad=0):
    return dict(name=name, op="quantise", rows=rows, n=n, dtype=dtype, pad=pad)


def _product(name, rows, vocab, n, cap=0.0, packed=False):
    return dict(name=name, op="logits", rows=rows, vocab=vocab, n=n, cap=cap, packed=packed)


def _select(name, groups, beams, vocab, n_out=None, history=0, rep=1.0, freq=0.0, pres=0.0, allowed=0.0, done=0.0,
            alpha=0.0, packed=False):
    return dict(name=name, op="select", groups=groups, beams=beams, vocab=vocab, n_out=n_out or beams, history=history,
                rep=rep, freq=freq, pres=pres, allowed=allowed, done=done, alpha=alpha, packed=packed)


def _reorder(name, groups, beams, layers, heads, room, length, width, dtype="bf16", history=0, keep=512):
    return dict(name=name, op="reorder", groups=groups, beams=beams, layers=layers, heads=heads, room=room,
                length=length, width=width, dtype=dtype, history=history, keep=keep)


def listed():
    return [
        # one token's hidden state before the LM head: latency alone
        _quantise("quantise 1x4096 bf16", 1, 4096, "bf16"),
        # an LM head's weights, a scale for each channel, when a model is loaded
        _quantise("quantise 50257x4096 f32", 50257, 4096, "f32"),
        # one token of a small model
        _product("logits 1x32000x2048", 1, 32000, 2048),
        # a decode step of a small batch: the weights are streamed once
        _product("logits 16x151936x4096", 16, 151936, 4096),
        # nothing is a multiple of anything: odd vocabulary, odd width, packed rows
        _product("logits 33x50257x2047", 33, 50257, 2047, packed=True),
        # a large decode step of a model with soft-capped logits
        _product("logits 512x262144x4096 cap", 512, 262144, 4096, cap=30.0),
        # one request of four beams
        _select("select 1x4x32000", 1, 4, 32000),
        # a serving batch with the sampler's penalties
        _select("select 16x4x151936", 16, 4, 151936, history=256, rep=1.15, freq=0.3, pres=0.5),
        # wide beams late in the search: finished beams compete by their normalised scores; packed rows of odd length
        _select("select 8x16x50257", 8, 16, 50257, done=0.25, alpha=0.8, packed=True),
        # a large constrained step: the allow-masks of a grammar
        _select("select 128x4x262144 masked", 128, 4, 262144, allowed=0.05),
        # a request's small states: grammar positions and histories, a one-layer cache
        _reorder("reorder 1x4 small", 1, 4, 1, 2, 64, 33, 64, history=200),
        # the caches of a serving batch: 16 requests of four beams
        _reorder("reorder 16x4 kv", 16, 4, 8, 8, 1024, 1000, 128, history=900, keep=1024),
    ]


MOST_PRODUCT = 512 * 262144 * 4096
MOST_WEIGHTS = 262144 * 4096
MOST_LOGITS = 512 * 262144
MOST_VALUES = 50257 * 4096
MOST_CACHE = 2 * 64 * 8 * 8 * 1000 * 128


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    odd = rng.random() < 0.3
    vocab = _log_int(rng, 32000, 262144)
    vocab = vocab | 1 if odd else (vocab + 63) // 64 * 64
    vocab = min(vocab, 262144)
    op = rng.choice(["quantise", "logits", "logits", "select", "select", "reorder"])
    if op == "quantise":
        n = _log_int(rng, 256, 8192)
        n = n | 1 if odd else (n + 15) // 16 * 16
        rows = min(_log_int(rng, 1, 50257), MOST_VALUES // n)
        c = _quantise("", rows, n, rng.choice(["bf16", "f16", "f32"]), pad=rng.choice([0, 0, 8]))
    elif op == "logits":
        n = _log_int(rng, 256, 8192)
        n = n | 1 if odd else (n + 15) // 16 * 16
        vocab = min(vocab, MOST_WEIGHTS // n)
        rows = max(1, min(_log_int(rng, 1, 512), MOST_PRODUCT // (n * vocab)))
        c = _product("", rows, vocab, n, cap=rng.choice([0.0, 0.0, 30.0]), packed=odd)
    elif op == "select":
        beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 12, 16])
        n_out = rng.choice([beams, beams, 2 * beams]) if beams > 1 else rng.randint(1, 8)
        groups = max(1, min(_log_int(rng, 1, 128), MOST_LOGITS // (beams * vocab), 512 // beams))
        history = rng.choice([0, _log_int(rng, 16, 1024)])
        done = rng.choice([0.0, 0.0, 0.25])
        c = _select("", groups, beams, vocab, n_out=n_out, history=history, rep=1.1 if history else 1.0,
                    freq=rng.choice([0.0, 0.2]) if history else 0.0, pres=rng.choice([0.0, 0.5]) if history else 0.0,
                    allowed=rng.choice([0.0, 0.0, 0.05, 0.3]), done=done, alpha=rng.choice([0.0, 0.6, 1.0]),
                    packed=odd)
    else:
        beams, groups = rng.choice([2, 3, 4, 5, 8, 12, 16]), _log_int(rng, 1, 32)
        room = _log_int(rng, 64, 2048)
        width = rng.choice([64, 80, 96, 128])
        heads = rng.choice([1, 2, 4, 8])
        layers = max(1, min(_log_int(rng, 1, 16), MOST_CACHE // (2 * groups * beams * heads * room * width)))
        groups = max(1, min(groups, MOST_CACHE // (2 * layers * beams * heads * room * width)))
        keep = rng.choice([64, 512, 1024])
        c = _reorder("", groups, beams, layers, heads, room, rng.randint(1, room), width,
                     dtype=rng.choice(["bf16", "f16", "f32"]), history=rng.randint(1, keep), keep=keep)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _hidden(case, g):
    """Hidden states or weights: rows of unlike size, a few entries far larger than the others (as hidden states
    after the last norm have), on rows of n + pad entries."""
    rows, n = case["rows"], case["n"]
    x = torch.randn((rows, n + case["pad"]), device=DEV, generator=g)
    x *= torch.exp(torch.randn((rows, 1), device=DEV, generator=g) * 0.5)
    far = torch.randint(0, n, (4,), device=DEV, generator=g)
    x[:, far] *= 8.0
    return x.to(DTYPES[case["dtype"]])


def _int8(rows, n, packed, g):
    """[rows, n] 8-bit values; the rows lie 16 bytes aligned unless packed."""
    ld = n if packed else (n + 15) // 16 * 16
    return torch.randint(-127, 128, (rows, ld), device=DEV, generator=g, dtype=torch.int8)[:, :n]


def _packed_bits(allow):
    """[rows, V] truth values as [rows, ceil(V / 32)] words, bit i % 32 of word i / 32."""
    rows, V = allow.shape
    W = (V + 31) // 32
    bits = torch.zeros((rows, W * 32), dtype=torch.bool, device=DEV)
    bits[:, :V] = allow
    w = (bits.view(rows, W, 32).long() << torch.arange(32, device=DEV)).sum(2)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def _select_inputs(case, seed):
    g = _gen(seed)
    rows, V, n = case["groups"] * case["beams"], case["vocab"], case["history"]
    ld = V if case["packed"] else (V + 63) // 64 * 64
    lg = torch.randn((rows, ld), device=DEV, generator=g) * 2.5
    likely = torch.randint(0, V, (rows, 32), device=DEV, generator=g)          # what the model would say next
    lg.scatter_add_(1, likely, 6.0 + 4.0 * torch.rand((rows, 32), device=DEV, generator=g))
    s = {"logits": lg[:, :V]}
    gap = 3.0 * torch.rand((case["groups"], case["beams"]), device=DEV, generator=g)
    s["scores"] = (-20.0 - gap.cumsum(1)).reshape(-1)
    if n:
        said = torch.randint(0, V, (rows, n), device=DEV, generator=g)
        again = likely.gather(1, torch.randint(0, 32, (rows, n), device=DEV, generator=g))
        pick = torch.rand((rows, n), device=DEV, generator=g) < 0.2
        s["hist_ids"] = torch.where(pick, again, said).int().reshape(-1)
        s["hist_off"] = torch.arange(rows + 1, device=DEV, dtype=torch.int32) * n
    if case["allowed"]:
        allow = torch.rand((rows, V), device=DEV, generator=g) < case["allowed"]
        allow.scatter_(1, likely[:, :8], True)
        if rows > 1:
            allow[1] = False                                                   # a beam whose grammar has ended
        s["mask"] = _packed_bits(allow)
    s["lengths"] = torch.full((rows,), 24, device=DEV, dtype=torch.int32)
    s["finished"] = None
    if case["done"]:
        over = torch.rand(rows, device=DEV, generator=g) < case["done"]
        s["finished"] = over.to(torch.uint8)
        s["lengths"] = torch.where(over, torch.randint(6, 24, (rows,), device=DEV, generator=g, dtype=torch.int32),
                                   s["lengths"])
    return s


def _parents(case, g):
    """Rows that survive a selection: the better beams of a group more often, ordered by nothing in particular."""
    groups, beams = case["groups"], case["beams"]
    u = torch.rand((groups, beams), device=DEV, generator=g)
    local = (u.square() * beams).int().clamp_(max=beams - 1)
    return (local + torch.arange(groups, device=DEV, dtype=torch.int32)[:, None] * beams).reshape(-1)


def _reorder_inputs(case, seed):
    g = _gen(seed)
    rows = case["groups"] * case["beams"]
    s = {"parents": _parents(case, g)}
    shape = (case["layers"], rows, case["heads"], case["room"], case["width"])
    s["keys"] = torch.randn(shape, device=DEV, generator=g, dtype=DTYPES[case["dtype"]])
    s["values"] = torch.randn(shape, device=DEV, generator=g, dtype=DTYPES[case["dtype"]])
    s["grammar"] = torch.randint(0, 256, (rows, GRAMMAR_ROW), device=DEV, generator=g, dtype=torch.uint8)
    s["tokens"] = torch.randint(0, 32000, (rows,), device=DEV, generator=g, dtype=torch.int32)
    lens = torch.randint(0, case["history"] + 1, (rows,), device=DEV, generator=g)
    off = torch.zeros(rows + 1, device=DEV, dtype=torch.int64)
    off[1:] = lens.cumsum(0)
    s["hist_off"] = off.int()
    s["hist_ids"] = torch.randint(0, 32000, (rows * case["history"],), device=DEV, generator=g, dtype=torch.int32)
    s["out_off"] = torch.zeros(rows + 1, device=DEV, dtype=torch.int32)
    s["out_ids"] = torch.zeros(rows * case["keep"], device=DEV, dtype=torch.int32)
    return s


def prepare(case, seed):
    op = case["op"]
    if op == "quantise":
        g = _gen(seed)
        s = {"x": _hidden(case, g)[:, :case["n"]]}
        s["q"] = torch.empty((case["rows"], case["n"]), dtype=torch.int8, device=DEV)
        s["scale"] = torch.empty(case["rows"], device=DEV)
    elif op == "logits":
        g = _gen(seed)
        rows, V, n = case["rows"], case["vocab"], case["n"]
        s = {"x": _int8(rows, n, case["packed"], g), "w": _int8(V, n, case["packed"], g)}
        # logits of a spread of about three
        s["x_scale"] = 0.02 * (0.5 + torch.rand(rows, device=DEV, generator=g))
        s["w_scale"] = 3.0 / (0.02 * 5400.0 * math.sqrt(n)) * (0.5 + torch.rand(V, device=DEV, generator=g))
        ld = V if case["packed"] else (V + 63) // 64 * 64
        s["logits"] = torch.zeros((rows, ld), device=DEV)[:, :V]
    elif op == "select":
        s = _select_inputs(case, seed)
        rows = case["groups"] * case["n_out"]
        s["out"] = {k: torch.empty(rows, device=DEV, dtype=t) for k, t in
                    (("tokens", torch.int32), ("parents", torch.int32), ("scores", torch.float32),
                     ("lengths", torch.int32), ("finished", torch.uint8))}
    else:
        s = _reorder_inputs(case, seed)
    s["case"] = case
    return s


# ---- one pass --------------------------------------------------------------------

def _plain_quantise(s):
    x = s["x"].float()
    # (64 bits: a quotient next to a half, and a scale's own rounding, decide whole steps)
    scale = (x.abs().amax(1, keepdim=True).double() / 127.0).float()
    q = torch.round(x.double() / scale.double())
    return {"values": q.float() * scale}


def _plain_logits(s):
    cap = s["case"]["cap"]
    y = s["x"].float() @ s["w"].float().t()
    y = y * s["x_scale"][:, None] * s["w_scale"]
    if cap > 0:
        y = cap * torch.tanh(y / cap)
    s["logits"].copy_(y)
    return {"logits": s["logits"]}


def _plain_select(s):
    """In 64 bits: the order of the candidates hangs on differences of long sums."""
    c = s["case"]
    groups, beams, V, n = c["groups"], c["beams"], c["vocab"], c["n_out"]
    rows, eos = groups * beams, c["vocab"] - 1
    lg = s["logits"].double()
    if "mask" in s:
        t = torch.arange(V, device=DEV)
        lg = torch.where((s["mask"][:, t >> 5] >> (t & 31)) & 1 == 1, lg, -math.inf)
    if "hist_ids" in s:
        ids = s["hist_ids"].view(rows, -1).long()
        count = torch.zeros_like(lg).scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float64))
        rep, freq, pres = (torch.tensor(c[k], dtype=torch.float32).double().item() for k in ("rep", "freq", "pres"))
        lg = torch.where(lg < 0, lg * rep ** count, lg / rep ** count)
        lg = lg - freq * count - pres * (count > 0)
    top = lg.amax(1, keepdim=True)
    z = torch.exp(lg - top).sum(1, keepdim=True)
    total = s["scores"].double()[:, None] + ((lg - top) - torch.log(z))
    total = torch.where(top > -math.inf, total, -math.inf)
    length = s["lengths"].double()[:, None] + 1.0
    if s["finished"] is not None:
        over = s["finished"].bool()[:, None]
        at_eos = torch.arange(V, device=DEV) == eos
        total = torch.where(over, torch.where(at_eos, s["scores"].double()[:, None], -math.inf), total)
        length = length - over.double()
    key = total / length.clamp(min=1.0) ** c["alpha"]
    best, at = torch.topk(key.view(groups, beams * V), min(n + 16, beams * V), dim=1)
    at, by_place = at.sort(1)                                    # equal keys: the lowest place first
    best, by_key = best.gather(1, by_place).sort(dim=1, descending=True, stable=True)
    best, at = best[:, :n], at.gather(1, by_key)[:, :n]
    fine = best > -math.inf
    row = at // V + torch.arange(groups, device=DEV)[:, None] * beams
    token = at % V
    over = token == eos
    score = total.view(groups, beams * V).gather(1, at)
    grown = length[:, 0][row]
    return {"tokens": torch.where(fine, token, -1).int().view(-1), "parents": torch.where(fine, row, -1).int().view(-1),
            "scores": torch.where(fine, score, -math.inf).float().view(-1),
            "lengths": torch.where(fine, grown, 0.0).int().view(-1), "finished": (fine & over).to(torch.uint8).view(-1)}


def _plain_reorder(s):
    c = s["case"]
    p = s["parents"].long()
    for k in ("keys", "values"):
        s[k][:, :, :, :c["length"]] = s[k][:, p, :, :c["length"]]
    s["grammar"].copy_(s["grammar"][p])
    # the histories, the new token appended, the last `keep` ids of each
    off = s["hist_off"].long()
    end, lens = off[1:][p], (off[1:] - off[:-1])[p]
    grown = (lens + 1).clamp(max=c["keep"])
    ends = grown.cumsum(0)
    s["out_off"][1:] = ends.int()
    place = torch.arange(s["out_ids"].numel(), device=DEV)
    row = torch.searchsorted(ends, place, right=True)
    used = row < p.numel()
    row = row.clamp(max=p.numel() - 1)
    back = ends[row] - place                                     # 1: the row's last entry
    old = s["hist_ids"][(end[row] + 1 - back).clamp(min=0, max=s["hist_ids"].numel() - 1)]
    s["out_ids"].copy_(torch.where(used, torch.where(back == 1, s["tokens"][row], old), s["out_ids"]))
    return {k: s[k] for k in ("keys", "values", "grammar", "out_off", "out_ids")}


def _own(s):
    from diskllm_amd import api
    c = s["case"]
    op = c["op"]
    if op == "quantise":
        q, scale = api.quantize_rows(s["x"], s["q"], s["scale"])
        return {"values": q * scale[:, None]}
    if op == "logits":
        return {"logits": api.logits_i8(s["x"], s["x_scale"], s["w"], s["w_scale"], softcap=c["cap"],
                                        out=s["logits"])}
    if op == "select":
        out = s["out"]
        api.beam_select(s["logits"], c["beams"], c["n_out"], scores=s["scores"], lengths=s["lengths"],
                        finished=s["finished"], hist_off=s.get("hist_off"), hist_ids=s.get("hist_ids"),
                        mask=s.get("mask"), eos_id=c["vocab"] - 1, length_penalty=c["alpha"],
                        repeat_penalty=c["rep"], frequency_penalty=c["freq"], presence_penalty=c["pres"],
                        max_history=c["history"], out=out)
        return out
    states = [api.beam_state(s["keys"], row_dim=1, length_dim=3, length=c["length"]),
              api.beam_state(s["values"], row_dim=1, length_dim=3, length=c["length"]),
              api.beam_state(s["grammar"])]
    api.beam_reorder(s["parents"], c["beams"], c["beams"], states,
                     history=api.beam_history(s["hist_off"], s["hist_ids"], s["tokens"], c["keep"], s["out_off"],
                                              s["out_ids"]))
    return {k: s[k] for k in ("keys", "values", "grammar", "out_off", "out_ids")}


PLAIN = {"quantise": _plain_quantise, "logits": _plain_logits, "select": _plain_select, "reorder": _plain_reorder}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    op = case["op"]
    if op == "quantise":
        n = case["rows"] * case["n"]
        size = 4 if case["dtype"] == "f32" else 2
        # the 8-bit values and scales, and what they stand for
        return {"bytes": n * size + n + 4 * case["rows"] + 4 * n, "flops": 5 * n}
    if op == "logits":
        rows, V, n = case["rows"], case["vocab"], case["n"]
        return {"bytes": (rows + V) * n + 4 * (rows + V) + 4 * rows * V, "flops": 2 * rows * V * n}
    if op == "select":
        rows, V = case["groups"] * case["beams"], case["vocab"]
        b = 4 * rows * (1.0 - case["done"]) * V + rows * (9 + 4 * case["history"]) + 17 * case["groups"] * case["n_out"]
        if case["allowed"]:
            b += 4 * rows * ((V + 31) // 32)
        return {"bytes": b, "flops": 16 * rows * V}
    # a row whose parent is not itself is written, a row with such a child read
    rows, beams = case["groups"] * case["beams"], case["beams"]
    p = [math.sqrt((k + 1) / beams) - math.sqrt(k / beams) for k in range(beams)]
    moved = sum(1.0 - q for q in p) / beams
    needed = sum(1.0 - (1.0 - q) ** (beams - 1) for q in p) / beams
    size = 4 if case["dtype"] == "f32" else 2
    row_bytes = 2 * case["layers"] * case["heads"] * case["length"] * case["width"] * size + GRAMMAR_ROW
    b = rows * row_bytes * (moved + needed) + rows * (2 * 4 * min(case["history"] / 2 + 1, case["keep"]) + 16)
    return {"bytes": b, "flops": 0}


# ---- the same from the definitions, in 64 bits -------------------------------------

def _exact_quantise(case, s):
    x = s["x"].to(torch.float64)
    scale = torch.div(x.abs().max(dim=1).values, 127.0).to(torch.float32).to(torch.float64)
    t = x / scale.unsqueeze(1)
    low = torch.floor(t)
    half = t - low - 0.5
    up = (half > 0) | ((half == 0) & (low.remainder(2) == 1))    # to the nearest, halves to the even one
    return {"values": (low + up) * scale.unsqueeze(1)}


def _exact_logits(case, s):
    x, w = s["x"].to(torch.float64), s["w"].to(torch.float64)
    y = torch.matmul(x * s["x_scale"].to(torch.float64).unsqueeze(1), w.t().contiguous())
    y *= s["w_scale"].to(torch.float64)
    if case["cap"] > 0:
        e = torch.exp(-2.0 * (y.abs() / case["cap"]))
        y = case["cap"] * torch.sign(y) * (1.0 - e) / (1.0 + e)
    return {"logits": y}


def _exact_select(case, s):
    """Group by group over the whole sorted list of its continuations."""
    beams, V, n = case["beams"], case["vocab"], case["n_out"]
    f = {k: float(torch.tensor(case[k], dtype=torch.float32)) for k in ("rep", "freq", "pres")}
    out = {"scores": []}
    for g in range(case["groups"]):
        sums, keys = [], []
        for r in range(g * beams, (g + 1) * beams):
            x = s["logits"][r].to(torch.float64)
            if "mask" in s:
                word = s["mask"][r].repeat_interleave(32)[:V]
                x = x.masked_fill((word >> torch.arange(V, device=DEV).remainder(32)).remainder(2) == 0, -math.inf)
            if "hist_ids" in s:
                a, b = int(s["hist_off"][r]), int(s["hist_off"][r + 1])
                ids, times = torch.unique(s["hist_ids"][a:b].long(), return_counts=True)
                v = x[ids]
                v = torch.where(v > 0, v / f["rep"] ** times, v * f["rep"] ** times)
                x[ids] = v - f["freq"] * times - f["pres"]
            over = s["finished"] is not None and bool(s["finished"][r])
            length = max(1, int(s["lengths"][r]) + (0 if over else 1))
            if over:
                x = torch.full_like(x, -math.inf)
                x[V - 1] = 0.0
                lse = 0.0
            else:
                lse = torch.logsumexp(x, 0)
            total = torch.where(x == -math.inf, -math.inf, x - lse + s["scores"][r].to(torch.float64))
            sums.append(total)
            keys.append(total / float(length) ** case["alpha"])
        order = torch.sort(torch.cat(keys), descending=True, stable=True).indices[:n]
        out["scores"].append(torch.cat(sums)[order])
    return {"tokens": None, "parents": None, "scores": torch.cat(out["scores"]), "lengths": None, "finished": None}


def exact(case, seed):
    op = case["op"]
    if op == "reorder":
        return None                                              # nothing is computed: values are moved
    s = prepare(case, seed)
    return {"quantise": _exact_quantise, "logits": _exact_logits, "select": _exact_select}[op](case, s)
