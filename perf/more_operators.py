"""The LM head in 4 bits and the scoring of its answers, and what they are measured on.

  quantise   dlk_quantize_mx and dlk_dequantize_mx: blocks of 32 values with a power-of-two scale, in 4 or 6 bits, and
             the values they stand for
  embed      dlk_dequantize_mx by token ids: rows of a tied 4-bit table
  logits     dlk_logits_mx: the LM head's product with 4-bit weights and 4- or 6-bit hidden states, soft-cap
  logprobs   dlk_token_logprobs: log-probabilities of given tokens, entropy, the most likely alternatives
  grad       dlk_token_logprobs_grad: the logits' gradient of those log-probabilities and of the entropy

With `own` false `run` computes them in elementary torch operations, with `own` true through diskllm_amd.api.
"""
import math

import torch

own = False


def _quantise(name, rows, n, dtype, fmt):
    return dict(name=name, op="quantise", rows=rows, n=n, dtype=dtype, fmt=fmt)


def _embed(name, rows, vocab, n, dtype):
    return dict(name=name, op="embed", rows=rows, vocab=vocab, n=n, dtype=dtype)


def _product(name, rows, vocab, n, fmt, cap=0.0):
    return dict(name=name, op="logits", rows=rows, vocab=vocab, n=n, fmt=fmt, cap=cap)


def _logprobs(name, rows, vocab, dtype, given=1, top=0, allowed=0.0, temp=1.0, packed=False):
    return dict(name=name, op="logprobs", rows=rows, vocab=vocab, dtype=dtype, given=given, top=top, allowed=allowed,
                temp=temp, packed=packed)


def _grad(name, rows, vocab, dtype, given=1, entropy=True, allowed=0.0, temp=1.0, packed=False):
    return dict(name=name, op="grad", rows=rows, vocab=vocab, dtype=dtype, given=given, entropy=entropy,
                allowed=allowed, temp=temp, packed=packed)


def listed():
    return [
        # one token's hidden state before the LM head: latency alone
        _quantise("quantise 1x4096 bf16 fp6", 1, 4096, "bf16", "fp6"),
        # an LM head's weights when a model is loaded, rows that end inside a block
        _quantise("quantise 100001x4090 bf16 fp4", 100001, 4090, "bf16", "fp4"),
        # the embedding rows of a decode step's tokens, of a tied table
        _embed("embed 16x4096", 16, 151936, 4096, "bf16"),
        # those of a batch of prompts
        _embed("embed 8192x4096 f32", 8192, 151936, 4096, "f32"),
        # one token of a small model
        _product("logits 1x32000x2048 fp4", 1, 32000, 2048, "fp4"),
        # a decode step of a small batch, hidden states in 6 bits: the weights are streamed once
        _product("logits 16x151936x4096 fp6", 16, 151936, 4096, "fp6"),
        # a large decode step of a model with soft-capped logits
        _product("logits 512x262144x4096 cap", 512, 262144, 4096, "fp4", cap=30.0),
        # one sampled token and its alternatives, as a chat request asks for them
        _logprobs("logprobs 1x32000 top 20", 1, 32000, "f32", top=20),
        # a decode step of a serving batch under grammar masks, packed rows of odd length
        _logprobs("logprobs 64x151937 masked", 64, 151937, "f32", given=1, top=5, allowed=0.3, temp=0.7, packed=True),
        # a prompt's tokens scored, with alternatives
        _logprobs("logprobs 2048x151936 bf16", 2048, 151936, "bf16", given=1, top=5),
        # a small policy-gradient step with an entropy bonus, several given tokens a row
        _grad("grad 48x50257 f32", 48, 50257, "f32", given=4, packed=True),
        # a batch of sequences' tokens in training
        _grad("grad 2048x151936 bf16", 2048, 151936, "bf16"),
    ]


MOST_VALUES = 100001 * 4090
MOST_EMBEDDED = 8192 * 4096
MOST_PRODUCT = 512 * 262144 * 4096
MOST_WEIGHTS = 262144 * 4096
MOST_LOGITS = 2048 * 151936


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    odd = rng.random() < 0.3
    vocab = _log_int(rng, 32000, 262144)
    vocab = min(vocab | 1 if odd else (vocab + 63) // 64 * 64, 262144)
    n = _log_int(rng, 256, 8192)
    n = n | 1 if odd else (n + 31) // 32 * 32
    op = rng.choice(["quantise", "embed", "logits", "logits", "logprobs", "logprobs", "grad"])
    if op == "quantise":
        rows = min(_log_int(rng, 1, 100001), MOST_VALUES // n)
        c = _quantise("", rows, n, rng.choice(["bf16", "f16", "f32"]), rng.choice(["fp4", "fp4", "fp6"]))
    elif op == "embed":
        vocab = min(vocab, MOST_WEIGHTS // n)
        rows = min(_log_int(rng, 1, 8192), MOST_EMBEDDED // n)
        c = _embed("", rows, vocab, n, rng.choice(["bf16", "f16", "f32"]))
    elif op == "logits":
        vocab = min(vocab, MOST_WEIGHTS // n)
        fmt = rng.choice(["fp4", "fp6"])
        rows = max(1, min(_log_int(rng, 1, 512), MOST_PRODUCT // (n * vocab)))
        c = _product("", rows, vocab, n, fmt, cap=rng.choice([0.0, 0.0, 30.0]))
    else:
        dtype = rng.choice(["bf16", "f16", "f32"])
        rows = max(1, min(_log_int(rng, 1, 2048), MOST_LOGITS // (vocab * (2 if dtype == "f32" else 1))))
        given = rng.choice([1, 1, 1, 2, 5, 16])
        allowed, temp = rng.choice([0.0, 0.0, 0.05, 0.3]), rng.choice([1.0, 1.0, 0.6, 1.5])
        if op == "logprobs":
            c = _logprobs("", rows, vocab, dtype, given, rng.choice([0, 1, 5, 20, 32]), allowed, temp, packed=odd)
        else:
            c = _grad("", rows, vocab, dtype, given, rng.random() < 0.6, allowed, temp, packed=odd)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
DEV = "cuda"
GRIDS = {"fp4": (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0),
         "fp6": tuple(i / 8 for i in range(16)) + tuple(i / 4 for i in range(8, 16)) + tuple(i / 2 for i in range(8, 16))}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _hidden(rows, n, g):
    """Hidden states or weights: rows of unlike size, a few entries far larger than the others (as hidden states
    after the last norm have)."""
    x = torch.randn((rows, n), device=DEV, generator=g)
    x *= torch.exp(torch.randn((rows, 1), device=DEV, generator=g) * 0.5)
    far = torch.randint(0, n, (4,), device=DEV, generator=g)
    x[:, far] *= 8.0
    return x


def _table(rows, n, g):
    """4-bit weights [rows, ceil(n / 32) * 16 bytes], scales [rows, ceil(n / 32)] on rows of whole 16 bytes."""
    blocks = (n + 31) // 32
    q = torch.randint(0, 256, (rows, blocks * 16), device=DEV, generator=g, dtype=torch.uint8)
    rest = n - (blocks - 1) * 32                             # the last block ends with zeros
    q[:, (blocks - 1) * 16 + (rest + 1) // 2:] = 0
    if rest % 2:
        q[:, (blocks - 1) * 16 + rest // 2] &= 15
    # logits of a spread of about three; blocks of unlike size
    e = 127 + round(math.log2(3.0 / (2.8 * 1.1 * math.sqrt(n))))
    scale = torch.randint(e - 1, e + 2, (rows, (blocks + 15) // 16 * 16), device=DEV, generator=g, dtype=torch.uint8)
    return q, scale[:, :blocks]


def _packed_bits(allow):
    """[rows, V] truth values as [rows, ceil(V / 32)] words, bit i % 32 of word i / 32."""
    rows, V = allow.shape
    W = (V + 31) // 32
    bits = torch.zeros((rows, W * 32), dtype=torch.bool, device=DEV)
    bits[:, :V] = allow
    w = (bits.view(rows, W, 32).int() << torch.arange(32, device=DEV, dtype=torch.int32)).sum(2, dtype=torch.int64)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def _scored(case, seed):
    g = _gen(seed)
    rows, V = case["rows"], case["vocab"]
    ld = V if case["packed"] else (V + 63) // 64 * 64
    lg = torch.empty((rows, ld), device=DEV, dtype=DTYPES[case["dtype"]])
    likely = torch.randint(0, V, (rows, 32), device=DEV, generator=g)          # what the model would say next
    for r in range(0, rows, 256):
        part = torch.randn((min(256, rows - r), ld), device=DEV, generator=g) * 2.5
        part.scatter_add_(1, likely[r:r + 256], 6.0 + 4.0 * torch.rand(likely[r:r + 256].shape, device=DEV, generator=g))
        lg[r:r + 256] = part
    s = {"logits": lg[:, :V]}
    pick = torch.randint(0, 32, (rows, case["given"]), device=DEV, generator=g)
    rare = torch.randint(0, V, (rows, case["given"]), device=DEV, generator=g)
    tokens = torch.where(torch.rand(rare.shape, device=DEV, generator=g) < 0.2, rare, likely.gather(1, pick))
    # (a prompt's padding)
    tokens = torch.where(torch.rand((rows, 1), device=DEV, generator=g) < 0.03, -1, tokens)
    s["tokens"] = tokens.int()
    if case["allowed"]:
        allow = torch.rand((rows, V), device=DEV, generator=g) < case["allowed"]
        allow.scatter_(1, likely[:, :24], True)
        if rows > 1:
            allow[1] = False                                                   # a row whose grammar has ended
        s["mask"] = _packed_bits(allow)
    return s, g


def prepare(case, seed):
    op = case["op"]
    if op == "quantise":
        s = {"x": _hidden(case["rows"], case["n"], _gen(seed)).to(DTYPES[case["dtype"]])}
    elif op == "embed":
        g = _gen(seed)
        s = dict(zip(("w", "w_scale"), _table(case["vocab"], case["n"], g)))
        s["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), device=DEV, generator=g, dtype=torch.int32)
    elif op == "logits":
        g = _gen(seed)
        s = dict(zip(("w", "w_scale"), _table(case["vocab"], case["n"], g)))
        s["x"], s["x_scale"] = _encode(_hidden(case["rows"], case["n"], g), case["fmt"])
        ld = (case["vocab"] + 63) // 64 * 64
        s["logits"] = torch.zeros((case["rows"], ld), device=DEV)[:, :case["vocab"]]
    else:
        s, g = _scored(case, seed)
        if op == "grad":
            rows = case["rows"]
            s["stats"] = torch.cat([_stats(s, case, r)[0] for r in range(0, rows, CHUNK)])
            s["grad_logprobs"] = torch.randn((rows, case["given"]), device=DEV, generator=g)
            s["grad_entropy"] = -0.01 * torch.rand(rows, device=DEV, generator=g) if case["entropy"] else None
            s["grad"] = torch.empty_strided(s["logits"].shape, s["logits"].stride(), dtype=s["logits"].dtype, device=DEV)
    s["case"] = case
    return s


# ---- one pass --------------------------------------------------------------------

CHUNK = 128               # rows that a plain form takes at once


def _times2(x, e):
    """x * 2^e (float64), e integers within +-1000: the power by its bits, as pow's own roundings show here."""
    return x * ((e.long() + 1023) << 52).view(torch.float64)


def _blocks(x):
    """x [rows, n] as float64 blocks [rows, blocks, 32], zeros behind n, and the exponent of each block's scale."""
    rows, n = x.shape
    b = torch.zeros((rows, (n + 31) // 32 * 32), dtype=torch.float64, device=x.device)
    b[:, :n] = x
    b = b.view(rows, -1, 32)
    top = b.abs().amax(2, keepdim=True)
    return b, torch.where(top > 0, torch.frexp(top).exponent - 1, -1000)


def _rounded(x, fmt):
    """The values that x [rows, n] is held as, and the exponents of its blocks' scales."""
    b, e = _blocks(x)
    e = (e - 2).clamp(-127, 127)
    t = _times2(b, -e)
    bits, most = (1, 6.0) if fmt == "fp4" else (3, 7.5)
    step = (torch.frexp(t).exponent - 1).clamp(min=0) - bits
    t = _times2(torch.round(_times2(t, -step)), step).clamp(-most, most)
    return t, e


def _encode(x, fmt):
    """x in the layout of dlk_quantize_mx: bytes and scales."""
    t, e = _rounded(x, fmt)
    rows, blocks = t.shape[:2]
    grid = torch.tensor(GRIDS[fmt], dtype=torch.float64, device=DEV)
    code = torch.bucketize(t.abs(), grid) + len(grid) * (t < 0)
    if fmt == "fp4":
        code = code.view(rows, -1, 2)
        q = (code[..., 0] + 16 * code[..., 1]).to(torch.uint8)
    else:
        code = code.view(rows, -1, 4)                        # four values in three bytes, the first lowest
        word = code[..., 0] + (code[..., 1] << 6) + (code[..., 2] << 12) + (code[..., 3] << 18)
        held = torch.stack((word & 255, word >> 8 & 255, word >> 16), 2).to(torch.uint8).view(rows, -1)
        q = torch.zeros((rows, (blocks * 24 + 15) // 16 * 16), dtype=torch.uint8, device=DEV)
        q[:, :blocks * 24] = held
        q = q[:, :blocks * 24]
    scale = torch.zeros((rows, (blocks + 15) // 16 * 16), dtype=torch.uint8, device=DEV)
    scale[:, :blocks] = (e + 127).squeeze(2)
    return q, scale[:, :blocks]


def _plain_quantise(s):
    x = s["x"]
    out = torch.empty_like(x)
    for r in range(0, x.shape[0], 8192):
        t, e = _rounded(x[r:r + 8192], s["case"]["fmt"])
        out[r:r + 8192] = _times2(t, e).view(t.shape[0], -1)[:, :x.shape[1]]
    return {"values": out}


def _decode(q, scale):
    """Float32 values of rows of blocks."""
    rows, blocks = scale.shape
    if q.shape[1] == blocks * 16:
        code, grid = torch.stack((q & 15, q >> 4), dim=2).int(), GRIDS["fp4"]
    else:
        b = q.reshape(rows, -1, 3).int()
        word = (b[..., 0] + (b[..., 1] << 8) + (b[..., 2] << 16)).unsqueeze(2)
        code, grid = word >> torch.tensor((0, 6, 12, 18), device=DEV) & 63, GRIDS["fp6"]
    v = torch.tensor(grid + tuple(-f for f in grid), device=DEV)[code]
    # (a scale's bits are a float's exponent)
    by = torch.where(scale == 0, 2.0 ** -127, (scale.int() << 23).view(torch.float32))
    return (v.reshape(rows, blocks, 32) * by.unsqueeze(2)).view(rows, blocks * 32)


def _plain_embed(s):
    t = s["tokens"].long()
    v = _decode(s["w"][t], s["w_scale"][t])[:, :s["case"]["n"]]
    return {"rows": v.to(DTYPES[s["case"]["dtype"]])}


def _plain_logits(s):
    cap = s["case"]["cap"]
    x = _decode(s["x"], s["x_scale"])
    for v in range(0, s["case"]["vocab"], 65536):
        y = x @ _decode(s["w"][v:v + 65536], s["w_scale"][v:v + 65536]).t()
        if cap > 0:
            y = cap * torch.tanh(y / cap)
        s["logits"][:, v:v + 65536] = y
    return {"logits": s["logits"]}


def _allowed(s, case, r):
    """Rows r .. of the logits in 32 bits, -inf where the mask has 0."""
    lg = s["logits"][r:r + CHUNK].float()
    if "mask" in s:
        t = torch.arange(case["vocab"], device=DEV)
        lg = torch.where((s["mask"][r:r + CHUNK, t >> 5] >> (t & 31)) & 1 == 1, lg, -math.inf)
    return lg


def _stats(s, case, r):
    """[rows, 4]: maximum, sum of exp((l - max) / T), entropy, log-sum; and the shifted logits (64 bits: log(1 +
    little))."""
    lg = _allowed(s, case, r)
    top = lg.amax(1, keepdim=True)
    some = top > -math.inf
    d = torch.where(some, lg.double() - top.double(), -math.inf) / case["temp"]
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    h = torch.where(some, torch.log(z) - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / z, 0.0)
    lse = top.double() / case["temp"] + torch.log(z)
    return torch.cat((top.double(), z, h, lse), 1).float(), d - torch.log(z), lg


def _plain_logprobs(s):
    c = s["case"]
    rows, V, k = c["rows"], c["vocab"], c["top"]
    out = {"logprobs": [], "stats": [], "top_ids": [], "top_logprobs": []}
    for r in range(0, rows, CHUNK):
        stats, lp, lg = _stats(s, c, r)
        lp = torch.where(lg > -math.inf, lp, -math.inf)
        t = s["tokens"][r:r + CHUNK].long()
        out["logprobs"].append(torch.where((t >= 0) & (t < V), lp.gather(1, t.clamp(0, V - 1)), 0.0).float())
        out["stats"].append(stats)
        if k:
            # largest first, of equal ones the lower id: the float's order above the id's
            u = lg.view(torch.int32).long()
            key = torch.where(u < 0, -(u & 0x7fffffff), u) * 2 ** 32 + (V - 1 - torch.arange(V, device=DEV))
            at = torch.topk(key, k, dim=1).indices
            best = lp.gather(1, at)
            out["top_ids"].append(torch.where(best > -math.inf, at, -1).int())
            out["top_logprobs"].append(best.float())
    return {n: torch.cat(v) for n, v in out.items() if v}


def _plain_grad(s):
    c = s["case"]
    V = c["vocab"]
    for r in range(0, c["rows"], CHUNK):
        lg = _allowed(s, c, r)
        top, z, h, _ = (s["stats"][r:r + CHUNK, k:k + 1] for k in range(4))
        live = lg > -math.inf
        d = torch.where(live, (lg - top) / c["temp"], -math.inf)
        p = torch.exp(d) / z
        t = s["tokens"][r:r + CHUNK].long()
        ok = (t >= 0) & (t < V)
        t = t.clamp(0, V - 1)
        g = torch.where(ok & live.gather(1, t), s["grad_logprobs"][r:r + CHUNK], 0.0)
        w = g.sum(1, keepdim=True)
        if s["grad_entropy"] is not None:
            w = w + s["grad_entropy"][r:r + CHUNK, None] * (d - torch.log(z) + h)
        y = torch.where(p > 0, -p * w, 0.0).scatter_add_(1, t, g)
        s["grad"][r:r + CHUNK] = y / c["temp"]
    return {"grad": s["grad"]}


def _own(s):
    from diskllm_amd import api
    c = s["case"]
    op = c["op"]
    if op == "quantise":
        q, scale = api.quantize_mx(s["x"], c["fmt"])
        return {"values": api.dequantize_mx(q, scale, n=c["n"], dtype=s["x"].dtype)}
    if op == "embed":
        return {"rows": api.dequantize_mx(s["w"], s["w_scale"], n=c["n"], ids=s["tokens"], dtype=DTYPES[c["dtype"]])}
    if op == "logits":
        return {"logits": api.logits_mx(s["x"], s["x_scale"], s["w"], s["w_scale"], softcap=c["cap"], out=s["logits"])}
    if op == "logprobs":
        out = api.token_logprobs(s["logits"], s["tokens"], top=c["top"], mask=s.get("mask"), temperature=c["temp"])
        return {k: v for k, v in out.items() if k in ("logprobs", "stats", "top_ids", "top_logprobs") and v is not None}
    return {"grad": api.token_logprobs_grad(s["logits"], s["tokens"], s["stats"], s["grad_logprobs"],
                                            grad_entropy=s["grad_entropy"], mask=s.get("mask"), temperature=c["temp"],
                                            out=s["grad"])}


PLAIN = {"quantise": _plain_quantise, "embed": _plain_embed, "logits": _plain_logits, "logprobs": _plain_logprobs,
         "grad": _plain_grad}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    op, rows = case["op"], case["rows"]
    if op in ("quantise", "embed", "logits"):
        blocks = (case["n"] + 31) // 32
    if op == "quantise":
        n = rows * case["n"]
        held = rows * blocks * (17 if case["fmt"] == "fp4" else 25)
        # the values, the blocks, and what those stand for
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 2 * held, "flops": 6 * n}
    if op == "embed":
        return {"bytes": rows * (blocks * 17 + 4 + case["n"] * SIZE[case["dtype"]]), "flops": rows * case["n"]}
    if op == "logits":
        V = case["vocab"]
        x = rows * blocks * (17 if case["fmt"] == "fp4" else 25)
        return {"bytes": x + V * blocks * 17 + 4 * rows * V, "flops": 2 * rows * V * case["n"]}
    V = case["vocab"]
    b = rows * V * SIZE[case["dtype"]] + rows * (8 * case["given"] + 16)
    if case["allowed"]:
        b += 4 * rows * ((V + 31) // 32)
    if op == "logprobs":
        return {"bytes": b + 8 * rows * case["top"], "flops": 8 * rows * V}
    return {"bytes": b + rows * V * SIZE[case["dtype"]], "flops": 8 * rows * V}


# ---- the same from the definitions, in 64 bits -------------------------------------

def _powers():
    """2^-127 .. 2^127, exactly."""
    return torch.tensor([2.0 ** k for k in range(-127, 128)], dtype=torch.float64, device=DEV)


def _grid(fmt):
    """The magnitudes of an element format."""
    bits = 1 if fmt == "fp4" else 3
    v = []
    for code in range(4 << bits):
        ex, m = code >> bits, code & ((1 << bits) - 1)
        v.append(m / 2.0 ** bits if ex == 0 else (1 + m / 2.0 ** bits) * 2.0 ** (ex - 1))
    return torch.tensor(v, dtype=torch.float64, device=DEV)


def _exact_quantise(case, s):
    """Each value to the nearest of the grid times its block's scale, halves to the even code."""
    grid, powers = _grid(case["fmt"]), _powers()
    x = s["x"]
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    emax = 2
    for r in range(0, x.shape[0], 4096):
        for i in range(0, x.shape[1], 32 * 16):
            part = x[r:r + 4096, i:i + 512].to(torch.float64)
            full = torch.nn.functional.pad(part, (0, -part.shape[1] % 32)).unflatten(1, (-1, 32))
            big = full.abs().max(dim=2, keepdim=True).values
            unit = powers[(torch.searchsorted(powers, big, right=True) - 1 - emax).clamp(0, 254)]
            v = full.abs() / unit
            hi = torch.searchsorted(grid, v).clamp(max=len(grid) - 1)          # the first that is not below
            lo = (hi - 1).clamp(min=0)
            below, above = v - grid[lo], grid[hi] - v
            code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
            out[r:r + 4096, i:i + 512] = (torch.sign(full) * grid[code] * unit).flatten(1)[:, :part.shape[1]]
    return {"values": out}


def _exact_rows(q, scale):
    width = q.shape[1] * 8 // (scale.shape[1] * 32)          # bits of a value
    grid = _grid("fp%d" % width)
    bit = q.unsqueeze(2) >> torch.arange(8, device=DEV, dtype=torch.uint8) & 1
    bit = bit.reshape(q.shape[0], -1, width).to(torch.float64)
    code = (bit * torch.tensor([2.0 ** k for k in range(width)], dtype=torch.float64, device=DEV)).sum(2).long()
    half = 2 ** (width - 1)
    v = torch.where(code >= half, -1.0, 1.0) * grid[code % half]
    return v * _powers()[scale.long()].repeat_interleave(32, 1)


def _exact_embed(case, s):
    t = s["tokens"].tolist()
    parts = [_exact_rows(s["w"][t[i:i + 1024]], s["w_scale"][t[i:i + 1024]]) for i in range(0, len(t), 1024)]
    return {"rows": torch.cat(parts)[:, :case["n"]]}


def _exact_logits(case, s):
    x = _exact_rows(s["x"], s["x_scale"])
    y = torch.empty((case["rows"], case["vocab"]), dtype=torch.float64, device=DEV)
    for v in range(0, case["vocab"], 16384):
        y[:, v:v + 16384] = torch.matmul(x, _exact_rows(s["w"][v:v + 16384], s["w_scale"][v:v + 16384]).t().contiguous())
    if case["cap"] > 0:
        e = torch.exp(-2.0 * (y.abs() / case["cap"]))
        y = case["cap"] * torch.sign(y) * (1.0 - e) / (1.0 + e)
    return {"logits": y}


def _row64(case, s, r):
    """Rows r .. r + 63 over the temperature in 64 bits, -inf where the mask has 0."""
    x = s["logits"][r:r + 64].to(torch.float64) / case["temp"]
    if "mask" in s:
        word = s["mask"][r:r + 64].repeat_interleave(32, 1)[:, :case["vocab"]]
        x = x.masked_fill((word >> torch.arange(case["vocab"], device=DEV).remainder(32)).remainder(2) == 0, -math.inf)
    return x


def _exact_logprobs(case, s):
    out = {"logprobs": [], "stats": [], "top_logprobs": []}
    for r in range(0, case["rows"], 64):
        x = _row64(case, s, r)
        lse = torch.logsumexp(x, 1)
        ended = lse == -math.inf
        lp = torch.where(ended[:, None], -math.inf, x - lse[:, None])
        top = x.max(1).values
        t = s["tokens"][r:r + 64].long()
        out["logprobs"].append(torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0))))
        entropy = -torch.special.xlogy(torch.exp(lp), torch.exp(lp)).sum(1)
        z = torch.where(ended, 0.0, torch.exp(lse - top))
        out["stats"].append(torch.stack((top * case["temp"], z, entropy, lse), 1))
        out["top_logprobs"].append(lp.sort(1, descending=True).values[:, :case["top"]])
    out = {k: torch.cat(v) for k, v in out.items()}
    if not case["top"]:
        del out["top_logprobs"]
        return out
    return {"logprobs": out["logprobs"], "stats": out["stats"], "top_ids": None, "top_logprobs": out["top_logprobs"]}


def _exact_grad(case, s):
    grads = torch.empty((case["rows"], case["vocab"]), dtype=torch.float64, device=DEV)
    for r in range(0, case["rows"], 64):
        x = _row64(case, s, r)
        live = x > -math.inf
        some = live.any(1, keepdim=True)
        lp = torch.where(live, x - torch.logsumexp(x, 1, keepdim=True), 0.0)
        p = torch.where(live, torch.exp(lp), 0.0)
        y = torch.zeros_like(p)
        for j in range(case["given"]):
            t = s["tokens"][r:r + 64, j:j + 1].long()
            at = t.clamp(min=0)
            g = torch.where((t >= 0) & live.gather(1, at), s["grad_logprobs"][r:r + 64, j:j + 1].to(torch.float64), 0.0)
            y -= g * p
            y.scatter_add_(1, at, g)
        if s["grad_entropy"] is not None:
            entropy = -(p * lp).sum(1, keepdim=True)
            y -= s["grad_entropy"][r:r + 64, None].to(torch.float64) * p * (lp + entropy)
        grads[r:r + 64] = torch.where(some, y / case["temp"], 0.0)
    return {"grad": grads}


def exact(case, seed):
    s = prepare(case, seed)
    return {"quantise": _exact_quantise, "embed": _exact_embed, "logits": _exact_logits, "logprobs": _exact_logprobs,
            "grad": _exact_grad}[case["op"]](case, s)
