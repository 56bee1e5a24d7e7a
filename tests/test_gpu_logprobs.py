"""dlk_token_logprobs and dlk_token_logprobs_grad against plain forms in 64 bits."""
import math
import os
import re

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                        # half a step of float32, relative
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}         # (8 bits: half of 2^-7)


def delta(vocab, dtype):
    """How far the sum z may be off, relative.  A term 2^t is off by ln2 |t| times the roundings of t = (l - m) * c (three:
    the difference, c and the product) and by the exponential's own 2 steps; the mean of ln2 |t| over the terms is at
    most ln V, as the entropy, log z plus that mean, is.  What a term is lowered by as maxima rise adds up to its |t|:
    the same again.  Each batch's lowering and those of waves, workgroup and row have an exponential's 2 steps (4 U)
    each; a batch adds 8 terms one after another and their 4 sums: 10 U."""
    batches = -(-vocab // (4096 if dtype == torch.float32 else 8192))
    return U * (6 * math.log(max(vocab, 2)) + 4 + 10 + 4 * (batches + 3))


def allow_words(allow):
    rows, V = allow.shape
    W = (V + 31) // 32
    bits = torch.zeros((rows, W * 32), dtype=torch.int64)
    bits[:, :V] = allow.cpu().long()
    w = (bits.view(rows, W, 32) << torch.arange(32)).sum(2)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int().to(allow.device)


def plain(logits, tokens, top, allow=None, T=1.0):
    """float64 (logprobs, stats, top ids, top logprobs, log p)."""
    T = float(torch.tensor(T, dtype=torch.float32))
    x = logits.double().cpu()
    if allow is not None:
        x = torch.where(allow.cpu(), x, -math.inf)
    bad = (x.isnan() | (x == math.inf)).any(1, keepdim=True)
    most = x.amax(1, keepdim=True)
    some = most > -math.inf
    d = torch.where(some, (x - most) / T, torch.tensor(-math.inf, dtype=torch.float64))
    d = torch.where(x == -math.inf, -math.inf, d)
    z = torch.exp(d).sum(1, keepdim=True)
    lp = d - torch.log(z)
    lp = torch.where(some, lp, -math.inf)
    e = torch.exp(lp)
    H = -torch.where(e > 0, e * lp, 0.0).sum(1, keepdim=True)
    stats = torch.cat((most, z, H, torch.where(some, most / T + torch.log(z), -math.inf)), 1)
    nan = torch.tensor(math.nan, dtype=torch.float64)
    stats = torch.where(bad, nan, stats)
    V = x.shape[1]
    out = torch.zeros(0)
    if tokens is not None:
        t = tokens.long().cpu()
        there = (t >= 0) & (t < V)
        out = torch.where(there, torch.where(bad, nan, lp.gather(1, t.clamp(0, V - 1))), 0.0)
    ids = tl = None
    if top:
        order = torch.sort(torch.where(x.isnan(), -math.inf, x), dim=1, descending=True, stable=True).indices[:, :top]
        tl = lp.gather(1, order)
        ids = torch.where(bad | (tl == -math.inf) & ~(x.gather(1, order) > -math.inf), -1, order)
        tl = torch.where(bad, nan, tl)
        if order.shape[1] < top:
            k = top - order.shape[1]
            ids = torch.nn.functional.pad(ids, (0, k), value=-1)
            tl = torch.cat((tl, torch.where(bad, nan, torch.tensor(-math.inf, dtype=torch.float64)).expand(-1, k)), 1)
    return out, stats, ids, tl, lp


def near(got, want, tol):
    got = got.double().cpu()
    # (a value past the type's largest, as -6.8e38 of two floats' ends, is an infinity there)
    same = (got == want.float().double()) | (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    assert (same | (off <= tol)).all(), (got, want, off.nan_to_num().max())


def check(logits, tokens, top=0, allow=None, T=1.0, words=None, mask_row=None, **kw):
    from diskllm_amd import api
    mask = words if words is not None else None if allow is None else allow_words(allow)
    got = api.token_logprobs(logits, tokens, top=top, mask=mask, mask_row=mask_row, temperature=T, **kw)
    torch.cuda.synchronize()
    lp, stats, ids, tl, _ = plain(logits, tokens if tokens is None or tokens.dim() == 2 else tokens[:, None], top, allow, T)
    V = logits.shape[1]
    d = delta(V, logits.dtype)
    if tokens is not None:
        near(got["logprobs"].view(lp.shape), lp, d + U * lp.abs())
    H, lse = stats[:, 2], stats[:, 3]
    near(got["stats"][:, 0], stats[:, 0], 0)
    near(got["stats"][:, 1], stats[:, 1], (d + U) * stats[:, 1])
    near(got["stats"][:, 2], H, d * (2 * math.log(max(V, 2)) + 2) + U * H)
    near(got["stats"][:, 3], lse, d + U * lse.abs())
    if top:
        assert torch.equal(got["top_ids"].cpu().long(), ids)
        near(got["top_logprobs"], tl, d + U * tl.abs())
    return got


def some(rows, V, dtype="f32", given=1, seed=0, spread=2.5, pad=0):
    g = torch.Generator("cuda").manual_seed(seed)
    lg = (torch.randn((rows, V + pad), device="cuda", generator=g) * spread).to(DTYPES[dtype])[:, :V]
    tokens = torch.randint(0, V, (rows, given), device="cuda", generator=g, dtype=torch.int32)
    return lg, tokens, g


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V,given,top", [
    (1, 1, 1, 1), (3, 2, 3, 5), (2, 7, 1, 64), (5, 100, 64, 3), (1, 4096, 1, 20), (3, 4097, 2, 64), (2, 8191, 0, 1),
    (4, 8193, 1, 0), (1, 50257, 1, 20), (65, 12345, 1, 5), (2, 151936, 7, 64), (900, 3001, 1, 2), (801, 20000, 1, 7),
    (1, 262144, 1, 33)])
def test_scores(cuda, dtype, rows, V, given, top):
    lg, tokens, _ = some(rows, V, dtype, given, seed=V + rows, pad=V % 3)
    check(lg, tokens if given else None, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V", [(1, 33), (7, 9001), (70, 40000), (850, 5000)])
@pytest.mark.parametrize("T", [0.6, 1.7])
def test_masked(cuda, dtype, rows, V, T):
    """Masks with a row that allows nothing, one that allows one id, and NaN and infinities in places not allowed."""
    lg, tokens, g = some(rows, V, dtype, 3, seed=V, pad=1)
    allow = torch.rand((rows, V), device="cuda", generator=g) < 0.1
    allow[0] = False
    if rows > 1:
        allow[1] = False
        allow[1, V - 1] = True
        allow[2:, tokens[2:, 0].long()] = True
    junk = torch.rand((rows, V), device="cuda", generator=g)
    lg[~allow & (junk < 0.1)] = math.nan
    lg[~allow & (junk > 0.9)] = math.inf
    lg[~allow & (junk > 0.45) & (junk < 0.5)] = -math.inf
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(lg, tokens, 5, allow, T, status=status)
    assert status.item() == 0


def test_long_rows(cuda):
    """More batches than a workgroup keeps records of."""
    lg, tokens, _ = some(1, 17_000_001, "f32", 2)
    lg[0, ::1000] = lg[0].amax() + 1                             # ties at the top, far apart
    check(lg, tokens, 40)
    lg, tokens, _ = some(258, 270_001, "bf16", 1, spread=1.0)
    lg[7, 3::50_000] = 9.0
    check(lg[:8], tokens[:8], 5)
    import diskllm_amd.api as api
    few, all_rows = api.token_logprobs(lg[:8], tokens[:8], top=5), api.token_logprobs(lg, tokens, top=5)
    assert torch.equal(few["top_ids"], all_rows["top_ids"][:8])
    near(all_rows["logprobs"][:8], few["logprobs"].double().cpu(), 2 * delta(270_001, torch.bfloat16))


@pytest.mark.parametrize("dtype,what", [("f32", r"rounding and\s+\*?\s*(\S+) at most"), ("bf16", r"16 bits: ([^;\s]+);"),
                                        ("f16", r"16 bits: ([^;\s]+);")])
def test_the_header_s_bound(cuda, dtype, what):
    """What the header says of 262,144 logits a row is what delta() derives, and holds where every batch's maximum is above
    all before it, so that each one lowers the sums."""
    from diskllm_amd import api
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "diskllm_amd.h")
    said = float(re.search(what, open(header).read()).group(1))
    V = 262144
    assert 0.9 * said <= delta(V, DTYPES[dtype]) <= said
    lg, tokens, _ = some(300, V, dtype, 3, seed=8, spread=1.0)
    lg += (torch.arange(V, device="cuda") * (24.0 / V)).to(lg.dtype)
    got = api.token_logprobs(lg, tokens)["logprobs"][::50]
    want = plain(lg[::50], tokens[::50], 0)[0]
    near(got, want, said + U * want.abs())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V", [(3, 40_000), (300, 9_000), (2, 600_001)])
@pytest.mark.parametrize("bits", [True, False])
def test_fewer_allowed_than_alternatives(cuda, dtype, rows, V, bits):
    """Rows that allow nothing, the type's lowest value alone, or a few ids, masked by bits or by -inf."""
    lg, tokens, g = some(rows, V, dtype, 2, seed=V + rows)
    allow = torch.zeros((rows, V), dtype=torch.bool, device="cuda")
    lowest = torch.tensor([0, V // 2, V - 1], device="cuda")
    allow[1, lowest] = True
    lg[1, lowest] = torch.finfo(DTYPES[dtype]).min
    if rows > 2:
        allow[2:].scatter_(1, torch.randint(0, V, (rows - 2, 9), device="cuda", generator=g), True)
        allow[2:].scatter_(1, tokens[2:, :1].long(), True)
    if not bits:
        lg[~allow] = -math.inf
    check(lg, tokens, 20, allow if bits else None)


@pytest.mark.parametrize("dtype,V", [("f32", 270_001), ("f32", 800_003), ("bf16", 530_001), ("f16", 1_100_000)])
def test_long_rows_of_one_workgroup(cuda, dtype, V):
    """Rows of more batches than a workgroup keeps records of, one workgroup each: many alternatives, ties, few allowed
    ids, none."""
    from diskllm_amd import api
    rows, top = 257, 40
    lg, tokens, g = some(rows, V, dtype, 2, seed=V, spread=1.0)
    lg[3, 5::V // 90] = 11.0                                     # more of the same than there are alternatives
    lg[4] = 0.5
    lg[5, :V - 70] = -math.inf
    lg[6] = -math.inf
    lg[7, :] = -math.inf
    lg[7, V - 1] = 2.0
    lg[8] = torch.finfo(DTYPES[dtype]).min
    at = [0, 3, 4, 5, 6, 7, 8, rows - 1]
    allow = torch.rand((2, V), device="cuda", generator=g) < 0.5
    of = torch.arange(rows, device="cuda", dtype=torch.int32) % 2
    d = delta(V, DTYPES[dtype])
    for mask in (None, allow_words(allow)):
        got = api.token_logprobs(lg, tokens, top=top, mask=mask, mask_row=of)
        lp, stats, ids, tl, _ = plain(lg[at], tokens[at], top, None if mask is None else allow[of[at].long()])
        assert torch.equal(got["top_ids"][at].cpu().long(), ids)
        near(got["top_logprobs"][at], tl, d + U * tl.abs())
        near(got["logprobs"][at], lp, d + U * lp.abs())
        near(got["stats"][at, 1], stats[:, 1], (d + U) * stats[:, 1])
        near(got["stats"][at, 2], stats[:, 2], d * (2 * math.log(V) + 2) + U * stats[:, 2])


def test_mask_rows_shared(cuda):
    """mask_row names the mask of each row."""
    lg, tokens, g = some(6, 5000, "f32", 1)
    allow = torch.rand((2, 5000), device="cuda", generator=g) < 0.3
    row = torch.tensor([1, 0, 0, 1, 1, 0], dtype=torch.int32, device="cuda")
    check(lg, tokens, 4, allow[row.long()], words=allow_words(allow), mask_row=row)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(2, 300), (3, 30001), (1000, 9000)])
@pytest.mark.parametrize("kind", ["equal", "three", "rising", "falling", "block", "zeros"])
def test_ties_and_orders(cuda, dtype, rows, V, kind):
    """Equal logits (the lowest ids come first) and orders in which lists fill and their bounds rise all the way."""
    g = torch.Generator("cuda").manual_seed(V)
    if kind == "equal":
        lg = torch.full((rows, V), 1.5, device="cuda")
    elif kind == "three":
        lg = torch.randint(0, 3, (rows, V), device="cuda", generator=g).float()
    elif kind == "rising":
        lg = (torch.arange(V, device="cuda") * 1e-3).expand(rows, V).contiguous()
    elif kind == "falling":
        lg = (torch.arange(V, device="cuda") * -1e-3).expand(rows, V).contiguous()
    elif kind == "block":
        lg = torch.zeros((rows, V), device="cuda")
        lg[:, V // 2:V // 2 + 200] = 3.0
    else:
        lg = torch.where(torch.rand((rows, V), device="cuda", generator=g) < 0.5, 0.0, -0.0)
    tokens = torch.randint(0, V, (rows, 1), device="cuda", generator=g, dtype=torch.int32)
    for top in (1, 20, 64):
        check(lg.to(DTYPES[dtype]), tokens, top)


def test_far_values(cuda):
    """The type's lowest value as a mask, its ends beside one another, -inf, one logit, and sure tokens."""
    lo, hi = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    V = 6000
    lg = torch.randn((12, V), device="cuda")
    lg[0] = lo
    lg[1, 5:] = lo
    lg[2, :] = lo
    lg[2, 77] = hi
    lg[3] = -math.inf
    lg[4] = -math.inf
    lg[4, 5999] = -3.0
    lg[5, 100] = 40.0
    lg[6, 100] = 1e30
    lg[7] *= 1e30
    lg[8] = hi
    lg[9, ::2] = -math.inf
    lg[10] *= 1e-30
    lg[11] += 1e6
    tokens = torch.tensor([[0, 100, 5999]] * 12, dtype=torch.int32, device="cuda")
    for T in (1.0, 1e-30, 1e30, 0.01):
        check(lg, tokens, 8, T=T)


@pytest.mark.parametrize("rows,V", [(3, 100), (4, 70000), (900, 3000)])
def test_not_finite(cuda, rows, V):
    """Rows with NaN or +inf: NaN, the status bit, and no other row touched."""
    for what in (math.nan, math.inf):
        lg, tokens, _ = some(rows, V, "f32", 2)
        lg[1, V - 1] = what
        tokens[1, 0] = -1
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        check(lg, tokens, 3, status=status)
        assert status.item() == 8


def test_no_tokens(cuda):
    """Tokens outside the vocabulary count as none."""
    lg, tokens, _ = some(4, 1000, "bf16", 4)
    tokens[0] = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1, 1000], dtype=torch.int32)
    got = check(lg, tokens, 0)
    assert (got["logprobs"][0] == 0).all()


def test_same_result_each_time(cuda):
    """Rows of many workgroups, in whatever order they end."""
    from diskllm_amd import api
    lg, tokens, _ = some(5, 200001, "bf16", 1)
    first = api.token_logprobs(lg, tokens, top=50)
    for _ in range(20):
        again = api.token_logprobs(lg, tokens, top=50)
        for k, v in first.items():
            assert torch.equal(v, again[k]), k


def test_offsets_past_32_bits(cuda):
    """Rows more than 2^32 elements apart."""
    from diskllm_amd import api
    ld, V = 1_500_000_000, 5000
    room = torch.empty(3 * ld + V, dtype=torch.bfloat16, device="cuda")
    lg = torch.as_strided(room, (4, V), (ld, 1))
    lg.copy_(torch.randn((4, V), device="cuda"))
    tokens = torch.tensor([[1], [2], [3], [4999]], dtype=torch.int32, device="cuda")
    got = check(lg, tokens, 3)
    g, h = torch.ones((4, 1), device="cuda"), torch.ones(4, device="cuda")
    want = api.token_logprobs_grad(lg.contiguous(), tokens, got["stats"], g, grad_entropy=h)
    api.token_logprobs_grad(lg, tokens, got["stats"], g, grad_entropy=h, out=lg)
    assert torch.equal(lg, want)


# ---- the gradient ----------------------------------------------------------------

def plain_grad(logits, tokens, g, h, allow=None, T=1.0):
    """float64 gradient, and how far it may be off before its last rounding."""
    T = float(torch.tensor(T, dtype=torch.float32))
    _, stats, _, _, lp = plain(logits, None, 0, allow, T)
    V = logits.shape[1]
    p = torch.exp(lp)
    lp = torch.where(p > 0, lp, 0.0)
    z, H = stats[:, 1:2], stats[:, 2:3]
    y = torch.zeros_like(p)
    G = torch.zeros_like(H)
    if tokens is not None:
        t = tokens.long().cpu()
        ok = (t >= 0) & (t < V)
        if allow is not None:
            ok &= allow.cpu().gather(1, t.clamp(0, V - 1))
        w = torch.where(ok, g.double().cpu(), 0.0)
        G = w.sum(1, keepdim=True)
        y.scatter_add_(1, t.clamp(0, V - 1), w)
        size = w.abs().sum(1, keepdim=True)
    else:
        size = torch.zeros_like(H)
    hh = torch.zeros_like(H) if h is None else h.double().cpu()[:, None]
    live = stats[:, :1] > -math.inf
    y = torch.where(live, (y - p * (G + hh * (lp + H))) / T, 0.0)
    d = delta(V, logits.dtype)
    lnz = torch.log(z.clamp(min=1))
    # p: its exponent's three roundings (4 U of ln2 |t| = lnz - lp), the exponential, 1 / z and products, z itself;
    # its weight: z and the entropy as the forward call left them, sums of up to 64 values, four roundings
    weight = size + hh.abs() * (lp.abs() + H + lnz + 1)
    off = p / T * weight * (U * (4 * (lnz - lp) + 16 + 64) + 3 * d) + p / T * hh.abs() * d * (2 * math.log(max(V, 2)) + 2)
    off = off + U * 70 * torch.zeros_like(y).scatter_add_(1, tokens.long().cpu().clamp(0, V - 1), g.abs().double().cpu()) / T \
        if tokens is not None else off
    return y, off + 2.0 ** -126 * weight / T


def check_grad(logits, tokens, g, h, allow=None, T=1.0, out=None):
    from diskllm_amd import api
    mask = None if allow is None else allow_words(allow)
    st = api.token_logprobs(logits, tokens, mask=mask, temperature=T)["stats"]
    want, off = plain_grad(logits, tokens, g, h, allow, T)
    got = api.token_logprobs_grad(logits, tokens, st, g, grad_entropy=h, mask=mask, temperature=T, out=out)
    dt = logits.dtype
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    near(got, want, off + HALF[dt] * (want.abs() + off) + tiny)
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V,given,entropy", [
    (1, 1, 1, True), (2, 5, 3, True), (3, 100, 64, False), (4, 4096, 1, True), (2, 8195, 2, True), (1, 50257, 1, False),
    (40, 12001, 1, True), (3, 151936, 5, True), (2, 1000, 0, True), (700, 777, 1, False)])
def test_gradient(cuda, dtype, rows, V, given, entropy):
    lg, tokens, gen = some(rows, V, dtype, max(given, 1), seed=V, pad=V % 2)
    if given > 2:
        tokens[:, 1] = tokens[:, 0]                              # the same token twice
        tokens[0, 2] = -1
    g = torch.randn((rows, max(given, 1)), device="cuda", generator=gen)
    h = torch.randn(rows, device="cuda", generator=gen) if entropy else None
    check_grad(lg, tokens if given else None, g if given else None, h)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [0.7, 3.0])
def test_gradient_masked(cuda, dtype, T):
    """Ids that are not allowed get zeros whatever stands there, tokens among them count for nothing."""
    rows, V = 9, 5003
    lg, tokens, gen = some(rows, V, dtype, 3, seed=5)
    allow = torch.rand((rows, V), device="cuda", generator=gen) < 0.3
    allow[0] = False
    allow.scatter_(1, tokens[:, :1].long(), True)
    allow[0] = False
    allow.scatter_(1, tokens[:, 1:2].long(), False)
    lg[~allow & (torch.rand((rows, V), device="cuda", generator=gen) < 0.2)] = math.nan
    g, h = torch.randn((rows, 3), device="cuda", generator=gen), torch.randn(rows, device="cuda", generator=gen)
    got = check_grad(lg, tokens, g, h, allow, T)
    assert (got[~allow] == 0).all() and (got[0] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_in_place_and_strided(cuda, dtype):
    """Over the logits themselves the same bits; into other strides what lies between rows is left."""
    from diskllm_amd import api
    lg, tokens, gen = some(6, 9001, dtype, 2, pad=5)
    g, h = torch.randn((6, 2), device="cuda", generator=gen), torch.randn(6, device="cuda", generator=gen)
    room = torch.full((6, 9001 + 3), 7.0, device="cuda", dtype=lg.dtype)
    got = check_grad(lg, tokens, g, h, out=room[:, 1:9002])
    assert (room[:, 0] == 7).all() and (room[:, 9002:] == 7).all()
    st = api.token_logprobs(lg, tokens)["stats"]
    want = got.clone()
    assert api.token_logprobs_grad(lg, tokens, st, g, grad_entropy=h, out=lg) is lg
    assert torch.equal(lg, want)


def test_nothing_to_differentiate(cuda):
    """Padding: rows whose weights are 0 or that have no token get zeros, also where their logits are NaN; a row that
    counts keeps its NaN."""
    from diskllm_amd import api
    lg, tokens, _ = some(5, 3000, "f32", 1)
    lg[1:, 7] = math.nan
    tokens[1] = -1
    g = torch.tensor([1.0, 2.0, 0.0, 0.0, 1.0], device="cuda")[:, None]
    h = torch.tensor([0.0, 0.0, 0.0, 0.5, 0.0], device="cuda")
    st = api.token_logprobs(lg, tokens)["stats"]
    got = api.token_logprobs_grad(lg, tokens, st, g, grad_entropy=h)
    assert (got[1:3] == 0).all() and got[3:].isnan().all() and not got[0].isnan().any()
    got = api.token_logprobs_grad(lg, tokens, st, g)
    assert (got[1:4] == 0).all() and got[4].isnan().all()


def test_gradient_against_differences(cuda):
    """Central differences of the 64-bit function at single logits: their own error is below h^2 / 6 times a third
    derivative of at most 12 for weights up to 1 and V = 40, plus 2^-52 of values up to 10 over h."""
    from diskllm_amd import api
    lg, tokens, gen = some(2, 40, "f32", 2, spread=1.0)
    g = torch.rand((2, 2), device="cuda", generator=gen)
    h = torch.rand(2, device="cuda", generator=gen)
    st = api.token_logprobs(lg, tokens, temperature=0.8)["stats"]
    got = api.token_logprobs_grad(lg, tokens, st, g, grad_entropy=h, temperature=0.8).double().cpu()
    step = 1e-4

    def value(x):
        lp, stats, _, _, _ = plain(x, tokens, 0, None, 0.8)
        return (lp * g.double().cpu()).sum(1) + stats[:, 2] * h.double().cpu()
    _, off = plain_grad(lg, tokens, g, h, None, 0.8)
    for v in range(40):
        up, down = lg.double().clone(), lg.double().clone()
        up[:, v] += step
        down[:, v] -= step
        want = (value(up) - value(down)) / (2 * step)
        assert ((got[:, v] - want).abs() <= off[:, v] + U * want.abs() + 12 / 0.8 ** 3 * step ** 2 + 1e-10).all()


def minus_infinity(rows, V, dtype, given, seed):
    """Logits of which a third are -inf, tokens among them (the first of each row is one, the last row's all are), two the
    same where there are more than two; where they are finite."""
    lg, tokens, gen = some(rows, V, dtype, given, seed=seed, pad=V % 2)
    dead = torch.rand((rows, V), device="cuda", generator=gen) < 0.3
    if given > 2:
        tokens[:, 2] = tokens[:, 0]
    dead.scatter_(1, tokens[:, 1:].long(), False)
    dead.scatter_(1, tokens[:, :1].long(), True)
    dead[-1].scatter_(0, tokens[-1].long(), True)
    lg[dead] = -math.inf
    return lg, tokens, ~dead, gen


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V,given,entropy", [
    (1, 2, 1, True), (3, 100, 64, True), (2, 4097, 2, False), (5, 9001, 3, True), (3, 50257, 64, False), (300, 777, 1, True),
    (2, 151936, 64, True)])
def test_gradient_of_minus_infinity(cuda, dtype, rows, V, given, entropy):
    """-inf in the logits is a mask: tokens there count for nothing and ids there get zeros, as the same rows masked by
    bits to the bit; over the logits themselves too, whose tokens other workgroups' stores could reach first."""
    from diskllm_amd import api
    lg, tokens, live, gen = minus_infinity(rows, V, dtype, given, V + given)
    g = torch.randn((rows, given), device="cuda", generator=gen)
    h = torch.randn(rows, device="cuda", generator=gen) if entropy else None
    st = api.token_logprobs(lg, tokens)["stats"]
    got = api.token_logprobs_grad(lg, tokens, st, g, grad_entropy=h)
    want, off = plain_grad(lg, tokens, g, h, live)               # (the mask in the place of -inf)
    tiny = torch.finfo(lg.dtype).smallest_normal * torch.finfo(lg.dtype).eps
    near(got, want, off + HALF[lg.dtype] * (want.abs() + off) + tiny)
    assert (got[~live] == 0).all()
    bits = api.token_logprobs_grad(lg, tokens, st, g, grad_entropy=h, mask=allow_words(live))
    assert torch.equal(got, bits)
    for _ in range(3):
        over = torch.empty_strided(lg.shape, lg.stride(), dtype=lg.dtype, device="cuda").copy_(lg)
        assert api.token_logprobs_grad(over, tokens, st, g, grad_entropy=h, out=over) is over
        assert torch.equal(over, got)


def test_gradient_of_minus_infinity_and_nan(cuda):
    """A row whose statistics are NaN: NaN, but zeros where its logits are -inf, and everywhere if all that is to be
    differentiated lies there."""
    from diskllm_amd import api
    lg, _, _ = some(3, 9000, "f32", 1)
    lg[:, ::3] = -math.inf
    lg[1:, 7] = math.nan
    tokens = torch.tensor([[3, 5000], [3, 5000], [3, 8001]], dtype=torch.int32, device="cuda")
    g = torch.ones((3, 2), device="cuda")
    st = api.token_logprobs(lg, tokens)["stats"]
    out = api.token_logprobs_grad(lg, tokens, st, g)
    assert (out[:, ::3] == 0).all() and not out[0].isnan().any() and (out[2] == 0).all()
    rest = torch.ones(9000, dtype=torch.bool, device="cuda")
    rest[::3] = False
    assert out[1, rest].isnan().all()
    api.token_logprobs_grad(lg, tokens, st, g, out=lg)
    assert torch.equal(lg.nan_to_num(nan=7.0), out.nan_to_num(nan=7.0))


def test_gradient_of_minus_infinity_against_differences(cuda):
    """Central differences at the finite logits of the 64-bit value over the tokens that have one (their own error as in
    test_gradient_against_differences)."""
    from diskllm_amd import api
    lg, tokens, live, gen = minus_infinity(2, 40, "f32", 3, 4)
    g = torch.rand((2, 3), device="cuda", generator=gen)
    h = torch.rand(2, device="cuda", generator=gen)
    st = api.token_logprobs(lg, tokens, temperature=0.8)["stats"]
    got = api.token_logprobs_grad(lg, tokens, st, g, grad_entropy=h, temperature=0.8).double().cpu()
    step = 1e-4

    def value(x):
        lp, stats, _, _, _ = plain(x, tokens, 0, None, 0.8)
        return torch.where(lp > -math.inf, lp * g.double().cpu(), 0.0).sum(1) + stats[:, 2] * h.double().cpu()
    _, off = plain_grad(lg, tokens, g, h, live, 0.8)
    for v in range(40):
        up, down = lg.double().clone(), lg.double().clone()
        up[:, v] += step
        down[:, v] -= step
        want = (value(up) - value(down)) / (2 * step)
        assert ((got[:, v] - want).abs() <= off[:, v] + U * want.abs() + 3 * 12 / 0.8 ** 3 * step ** 2 + 1e-10).all()


def test_gradient_in_place_graph(cuda):
    """In place and captured: replays over new logits, eager calls between them."""
    from diskllm_amd import api
    rows, V, given = 4, 30001, 5
    src, tokens, _, gen = minus_infinity(rows, V, "f32", given, 9)
    g, h = torch.randn((rows, given), device="cuda", generator=gen), torch.randn(rows, device="cuda", generator=gen)
    over = torch.empty_like(src)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = api.token_logprobs(src, tokens)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            over.copy_(src)
            api.token_logprobs(over, tokens, out=out)
            api.token_logprobs_grad(over, tokens, out["stats"], g, grad_entropy=h, out=over)
        for k in range(4):
            src.copy_(torch.where(src > -math.inf, src + 0.25 * k, src).roll(17 * k, 1))
            graph.replay()
            st = api.token_logprobs(src, tokens)["stats"]
            want = api.token_logprobs_grad(src, tokens, st, g, grad_entropy=h)
            side.synchronize()
            assert torch.equal(over, want)
    side.synchronize()


def test_more_rows_than_a_launch(cuda):
    """2^24 rows and more, a workgroup each."""
    from diskllm_amd import api
    rows, V = (1 << 24) + 70_001, 3
    g = torch.Generator("cuda").manual_seed(2)
    lg = torch.randn((rows, V), device="cuda", generator=g)
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=g, dtype=torch.int32)
    got = api.token_logprobs(lg, tokens, top=1)
    w = torch.ones((rows, 1), device="cuda")
    grad = api.token_logprobs_grad(lg, tokens, got["stats"], w)
    d = delta(V, torch.float32)
    for a in range(0, rows, 1 << 22):
        s = slice(a, min(a + (1 << 22), rows))
        lp = torch.log_softmax(lg[s].double(), 1)
        want = lp.gather(1, tokens[s, None].long())[:, 0]
        assert ((got["logprobs"][s].double() - want).abs() <= d + U * want.abs()).all()
        first = torch.where(lg[s] == lg[s].amax(1, keepdim=True), torch.arange(V, device="cuda"), V).amin(1)
        assert torch.equal(got["top_ids"][s, 0].long(), first)
        p = lp.exp()
        want = torch.nn.functional.one_hot(tokens[s].long(), V) - p
        # (as plain_grad's, of one token of weight 1, and half a step of the result)
        off = p * (U * (4 * (math.log(V) - lp) + 80) + 3 * d) + U * 70
        assert ((grad[s].double() - want).abs() <= off + U * want.abs()).all()
    api.token_logprobs_grad(lg, tokens, got["stats"], w, out=lg)
    assert torch.equal(lg, grad)


# ---- streams, graphs, the path as a whole ------------------------------------------

def test_graph(cuda):
    """Captured with a sample and a beam step on one stream: replays with new logits, eager calls of other sizes (the same
    workspace) between them."""
    from diskllm_amd import api
    rows, V = 6, 30000
    lg, tokens, gen = some(rows, V, "f32", 1)
    g, h = torch.ones((rows, 1), device="cuda"), torch.full((rows,), 0.1, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = api.token_logprobs(lg, tokens, top=9)
        beams = api.beam_select(lg, 2, 2)
        grad = api.token_logprobs_grad(lg, tokens, out["stats"], g, grad_entropy=h)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            api.beam_select(lg, 2, 2, out=beams)
            api.token_logprobs(lg, tokens, top=9, out=out)
            api.token_logprobs_grad(lg, tokens, out["stats"], g, grad_entropy=h, out=grad)
        other, other_tokens, _ = some(3, 250000, "bf16", 1, seed=9)
        for k in range(4):
            lg.copy_(torch.randn((rows, V), device="cuda", generator=gen) * 3)
            graph.replay()
            api.token_logprobs(other, other_tokens, top=64)
            again = api.token_logprobs(lg, tokens, top=9)
            side.synchronize()
            for n in again:
                assert torch.equal(again[n], out[n])
            assert torch.equal(grad, api.token_logprobs_grad(lg, tokens, out["stats"], g, grad_entropy=h))
    side.synchronize()


def test_two_streams(cuda):
    """Calls on two streams at once have workspaces of their own."""
    from diskllm_amd import api
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    lg, tokens, _ = some(4, 200000, "f32", 1)
    lg2, tokens2, _ = some(4, 200000, "f32", 1, seed=1)
    want, want2 = api.token_logprobs(lg, tokens, top=30), api.token_logprobs(lg2, tokens2, top=30)
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        with torch.cuda.stream(a):
            x = api.token_logprobs(lg, tokens, top=30)
        with torch.cuda.stream(b):
            y = api.token_logprobs(lg2, tokens2, top=30)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        for k in want:
            assert torch.equal(x[k], want[k]) and torch.equal(y[k], want2[k])


def test_a_decode_step(cuda):
    """The path as it is used: hidden states in blocks, 4-bit head, greedy sample, its score, and the embedding of the
    drawn tokens from the tied table."""
    import numpy as np
    from diskllm_amd import api, workloads
    w = workloads.c1()
    V, n = w.vocab, 256
    g = torch.Generator("cuda").manual_seed(1)
    table, table_scale = api.quantize_mx(torch.randn((V, n), device="cuda", generator=g))
    hidden = torch.randn((1, n), device="cuda", generator=g).bfloat16()
    q, s = api.quantize_mx(hidden, "fp6")
    logits = api.logits_mx(q, s, table, table_scale, out=torch.empty((1, V), device="cuda"))
    w.logits, w.temperature, w.repeat_penalty, w.hist_off, w.hist_ids = logits.cpu().numpy(), 0.0, 1.0, None, None
    db = api.to_device(w)
    api.sample(db)
    got = api.token_logprobs(logits, db.out_ids, top=2)
    assert got["top_ids"][0, 0] == db.out_ids[0] == int(np.argmax(w.logits[0]))
    assert got["top_logprobs"][0, 0] == got["logprobs"][0]
    check(logits, db.out_ids, 2)
    e = api.dequantize_mx(table, table_scale, ids=db.out_ids, dtype=torch.bfloat16)
    assert torch.equal(e, api.dequantize_mx(table, table_scale, dtype=torch.bfloat16)[db.out_ids.long()])
    x = api.dequantize_mx(q, s).double()
    near(logits[0, db.out_ids.long()], (x @ api.dequantize_mx(table, table_scale)[db.out_ids.long()].double().t())[0].cpu(), 1e-4)
