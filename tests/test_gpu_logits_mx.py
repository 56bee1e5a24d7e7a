"""dlk_quantize_mx, dlk_dequantize_mx and dlk_logits_mx against plain forms in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GRID = {"fp4": np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6]),
        "fp6": np.array([i / 8 for i in range(16)] + [i / 4 for i in range(8, 16)] + [i / 2 for i in range(8, 16)])}
WIDTH = {"fp4": 16, "fp6": 24}


def pack(codes, fmt):
    """Bytes of codes [rows, blocks * 32]."""
    rows = codes.shape[0]
    bits = 4 if fmt == "fp4" else 6
    b = (codes[:, :, None] >> np.arange(bits)) & 1
    return np.packbits(b.reshape(rows, -1, 8).astype(np.uint8), axis=2, bitorder="little").reshape(rows, -1)


def codes_of(q, fmt):
    bits = 4 if fmt == "fp4" else 6
    b = np.unpackbits(q[:, :, None], axis=2, bitorder="little").reshape(q.shape[0], -1, bits)
    return (b.astype(np.int64) << np.arange(bits)).sum(2)


def values(q, scale, fmt):
    """float64 [rows, blocks * 32]."""
    c = codes_of(q, fmt)
    half = len(GRID[fmt])
    v = GRID[fmt][c % half] * np.where(c >= half, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return v * np.repeat(s, 32, 1)


def quantized(x, fmt):
    """(bytes, scales) of float64 rows as the header says."""
    rows, n = x.shape
    blocks = (n + 31) // 32
    b = np.zeros((rows, blocks * 32))
    b[:, :n] = x
    b = b.reshape(rows, blocks, 32)
    top = np.abs(b).max(2)
    bad = ~np.isfinite(top)
    e = np.frexp(np.where(bad | (top == 0), 2.0 ** -200, top))[1] - 1 - 2
    e = np.maximum(e, -127)
    with np.errstate(all="ignore"):
        t = np.ldexp(np.abs(b), -e[:, :, None])
    grid = GRID[fmt]
    hi = np.clip(np.searchsorted(grid, t), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    with np.errstate(all="ignore"):
        down, up = t - grid[lo], grid[hi] - t
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = np.where(bad[:, :, None], 0, code + len(grid) * (np.signbit(b) & ~bad[:, :, None]))
    return pack(code.reshape(rows, -1), fmt), np.where(bad, 255, e + 127).astype(np.uint8)


def check_quantized(torch, x, fmt, **kw):
    from diskllm_amd import api
    q, s = api.quantize_mx(x, fmt, **kw)
    torch.cuda.synchronize()
    want_q, want_s = quantized(x.double().cpu().numpy(), fmt)
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    return q, s


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,n,pad", [(1, 1, 0), (1, 31, 0), (3, 32, 3), (5, 33, 0), (70, 100, 1), (2, 1025, 0),
                                        (1, 4096, 0), (33, 2048, 8), (4, 8193, 1), (3000, 8, 0)])
def test_quantize(cuda, fmt, dtype, rows, n, pad):
    import torch
    g = torch.Generator("cuda").manual_seed(rows * 1000 + n)
    x = torch.randn((rows, n + pad), device="cuda", generator=g) * 3
    check_quantized(torch, x.to(getattr(torch, dtype))[:, :n], fmt)


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
def test_quantize_special_blocks(cuda, fmt):
    """Zeros, halves that go to the even code, saturation, NaN, infinities, the smallest and largest magnitudes."""
    import torch
    x = np.zeros((14, 64), np.float32)
    grid = GRID[fmt]
    mid = np.concatenate(((grid[1:] + grid[:-1]) / 2, [7.75, 7.0, 7.99]))
    for k, e in enumerate((0, 100, -120, -126)):                 # halves, and next to them on both sides
        t = np.concatenate((mid, np.nextafter(mid.astype(np.float32), 0), np.nextafter(mid.astype(np.float32), 9)))
        t = t.astype(np.float32)[:31 if k < 3 else 20]
        x[k, 0] = np.ldexp(np.float32(4.0), e)
        x[k, 1:1 + len(t)] = np.ldexp(t, e) * np.where(np.arange(len(t)) % 2, -1, 1)
        x[k, 32:32 + len(t)] = x[k, 1:1 + len(t)]
    x[4, 7], x[4, 40] = np.nan, -1.0
    x[5, 50], x[5, 3] = np.inf, 2.0
    x[6, 0] = -np.inf
    x[7] = np.float32(1e-45) * np.arange(64)
    x[8] = np.float32(1e-38) * np.linspace(-1, 1, 64)
    x[9] = np.float32(3.4e38) * np.linspace(-1, 1, 64)
    x[10] = -0.0
    x[11, 9] = np.float32(1e-45)
    x[12, :32] = np.float32(3e38)
    x[12, 32:] = np.float32(2.0 ** -125) * np.linspace(0.5, 2, 32)
    x[13, :5] = [2.0 ** 127, 2.0 ** 121, -2.0 ** 122, 2.0 ** 120, 3.0 * 2.0 ** 119]
    q, s = check_quantized(torch, torch.from_numpy(x).cuda(), fmt)
    assert s[4].tolist()[0] == 255 and s[4].tolist()[1] != 255 and s[10].tolist() == [0, 0]


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("top", [-126, -120, -60, -10, -3, 0, 3, 30, 100, 127])
def test_quantize_every_bfloat16(cuda, fmt, top):
    """Every bfloat16 up to a block's largest, whose exponent is `top`."""
    import torch
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    v = v[v.isfinite()]
    v = v[v.double().abs() < 2.0 ** (top + 1)]
    v = torch.cat((v, v.new_zeros(-len(v) % 31))).view(-1, 31)
    x = torch.cat((torch.full((len(v), 1), 2.0 ** top, dtype=torch.bfloat16), v), 1)
    check_quantized(torch, x.cuda(), fmt)


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
def test_quantize_into_strided(cuda, fmt):
    """Into rows of other strides; what lies between the rows is left."""
    import torch
    x = torch.randn((9, 100), device="cuda")
    width = 4 * WIDTH[fmt]
    q = torch.full((9, width + 24), 77, dtype=torch.uint8, device="cuda")
    s = torch.full((9 * 7 + 1,), 77, dtype=torch.uint8, device="cuda")
    check_quantized(torch, x, fmt, q=q[:, 8:8 + width], scale=s[1:].view(9, 7)[:, :4])
    assert (q[:, :8] == 77).all() and (q[:, 8 + width:] == 77).all()
    assert (s[1:].view(9, 7)[:, 4:] == 77).all() and s[0] == 77


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_dequantize_every_code(cuda, fmt, dtype):
    """Every code under small, usual, large and NaN scales, rounded once."""
    import torch
    from diskllm_amd import api
    codes = 2 * len(GRID[fmt])
    scales = np.array([0, 1, 2, 100, 110, 125, 127, 130, 140, 200, 253, 254, 255], np.uint8)
    c = np.tile(np.arange(64) % codes, (len(scales), 1))
    q, s = pack(c, fmt), np.stack((scales, scales[::-1]), 1)
    got = api.dequantize_mx(torch.from_numpy(q).cuda(), torch.from_numpy(s.copy()).cuda(), dtype=getattr(torch, dtype))
    with np.errstate(all="ignore"):
        want = torch.from_numpy(values(q, s, fmt)).to(getattr(torch, dtype))
    assert torch.equal(got.cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
    assert torch.equal(got.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("rows,n", [(1, 1), (7, 33), (40, 96), (5, 4096), (3, 2047), (2000, 9)])
def test_dequantize_rows(cuda, fmt, rows, n):
    """Rows as they are and by ids (repeated, outside the table), into strided rows."""
    import torch
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(n)
    q, s = api.quantize_mx(torch.randn((rows, n), device="cuda", generator=g), fmt)
    want = torch.from_numpy(values(q.cpu().numpy(), s.cpu().numpy(), fmt))[:, :n].float()
    assert torch.equal(api.dequantize_mx(q, s, n=n).cpu(), want)
    ids = torch.tensor([0, rows - 1, rows, -1, rows - 1, -2 ** 31, 2 ** 31 - 1, rows // 2], dtype=torch.int32, device="cuda")
    out = torch.full((8, n + 3), 7.0, device="cuda")
    api.dequantize_mx(q, s, n=n, ids=ids, out=out[:, 1:1 + n])
    at = torch.tensor([0, rows - 1, 0, 0, rows - 1, 0, 0, rows // 2])
    there = torch.tensor([1, 1, 0, 0, 1, 0, 0, 1])[:, None]
    assert torch.equal(out[:, 1:1 + n].cpu(), want[at] * there)
    assert (out[:, 0] == 7).all() and (out[:, 1 + n:] == 7).all()


def inputs(torch, rows, vocab, n, fmt, seed=0, spread=3):
    """Hidden states and weights in blocks, with junk behind the scales; their values."""
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(seed)
    def some(r, f):
        x = torch.randn((r, n), device="cuda", generator=g)
        x *= torch.exp2(torch.randint(-spread, spread + 1, (r, 1), device="cuda", generator=g).float())
        blocks = (n + 31) // 32
        scale = torch.full((r, (blocks + 15) // 16 * 16), 255, dtype=torch.uint8, device="cuda")
        return api.quantize_mx(x, f, scale=scale[:, :blocks])
    return some(rows, fmt) + some(vocab, "fp4")


def check_product(torch, x, xs, w, ws, fmt, softcap=0.0, out=None):
    """Off by at most 2^-22 of the products' sizes for each 128 values (added over the row's length, a zero sum's
    first step among them), and the cap as the header says."""
    from diskllm_amd import api
    got = api.logits_mx(x, xs, w, ws, softcap=softcap, out=out)
    X, W = (torch.from_numpy(values(a.cpu().numpy(), b.cpu().numpy(), f)) for a, b, f in ((x, xs, fmt), (w, ws, "fp4")))
    want = X @ W.t()
    tol = (X.abs() @ W.abs().t()) * (-(-X.shape[1] // 512) * 4) * 2.0 ** -22 + 2.0 ** -149
    if softcap > 0:
        want = softcap * torch.tanh(want / softcap)              # (1-Lipschitz in the product)
        tol = tol + want.abs() * 2.0 ** -20 + softcap * 2.0 ** -148
    off = (got.double().cpu() - want).abs()
    assert not off.isnan().any()
    assert (off <= tol).all(), (off - tol).max().item()
    return got


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("rows,vocab,n", [
    (1, 1, 1), (1, 64, 32), (2, 65, 33), (16, 63, 511), (17, 129, 512), (15, 200, 513), (32, 1000, 2047), (33, 257, 96),
    (64, 300, 1024), (65, 100, 1000), (128, 259, 4096), (129, 511, 256), (200, 256, 257), (385, 513, 640), (513, 300, 40),
    (256, 256, 256), (256, 300, 32), (257, 255, 512), (500, 1000, 288), (512, 257, 4128), (1000, 256, 33), (640, 520, 513),
    (1, 5000, 8192), (3, 70, 31)])
def test_product(cuda, fmt, rows, vocab, n):
    import torch
    check_product(torch, *inputs(torch, rows, vocab, n, fmt, seed=rows + n), fmt)


@pytest.mark.parametrize("rows", [1, 40, 400])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e-39, 1e30])
def test_product_capped(cuda, rows, cap):
    import torch
    check_product(torch, *inputs(torch, rows, 301, 200, "fp4", spread=0), "fp4", softcap=cap)


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("rows", [5, 150, 500])
def test_product_strided(cuda, fmt, rows):
    """Rows of larger strides; logits of any stride, what stands past the vocabulary left."""
    import torch
    vocab, n = 131, 300
    x, xs, w, ws = inputs(torch, rows, vocab, n, fmt)
    X = torch.full((rows, x.shape[1] + 32), 255, dtype=torch.uint8, device="cuda")
    X[:, 16:16 + x.shape[1]] = x
    W = torch.full((vocab, w.shape[1] + 48), 255, dtype=torch.uint8, device="cuda")
    W[:, 32:32 + w.shape[1]] = w
    room = torch.full((rows, vocab + 7), 5.0, device="cuda")
    check_product(torch, X[:, 16:16 + x.shape[1]], xs, W[:, 32:32 + w.shape[1]], ws, fmt, out=room[:, 3:3 + vocab])
    assert (room[:, :3] == 5).all() and (room[:, 3 + vocab:] == 5).all()


@pytest.mark.parametrize("rows,vocab,n", [(500, 301, 300), (256, 258, 1056), (300, 259, 600)])
@pytest.mark.parametrize("far", [False, True])
def test_product_of_many_rows_strided(cuda, rows, vocab, n, far):
    """Rows of hidden states, weights and scales apart (weights by 4 MB: past the offsets of one tile), logits in a
    larger matrix, at a place of its own in a row."""
    import torch
    x, xs, w, ws = inputs(torch, rows, vocab, n, "fp4")
    blocks = xs.shape[1]
    X = torch.full((rows, x.shape[1] + 32), 255, dtype=torch.uint8, device="cuda")
    X[:, 16:16 + x.shape[1]] = x
    W = torch.full((vocab, 1 << 22 if far else w.shape[1] + 48), 255, dtype=torch.uint8, device="cuda")
    W[:, 32:32 + w.shape[1]] = w
    XS = torch.full((rows, (blocks + 15) // 16 * 16 + 16), 255, dtype=torch.uint8, device="cuda")
    XS[:, 16:16 + blocks] = xs
    WS = torch.full((vocab, (blocks + 15) // 16 * 16 + 32), 255, dtype=torch.uint8, device="cuda")
    WS[:, 16:16 + blocks] = ws
    room = torch.full((rows + 1, vocab + 7), 5.0, device="cuda")
    check_product(torch, X[:, 16:16 + x.shape[1]], XS[:, 16:16 + blocks], W[:, 32:32 + w.shape[1]], WS[:, 16:16 + blocks],
                  "fp4", out=room[:rows, 3:3 + vocab])
    assert (room[:rows, :3] == 5).all() and (room[:rows, 3 + vocab:] == 5).all() and (room[rows] == 5).all()


def test_product_of_many_rows_is_each_rows_own(cuda):
    """Tiles that lie over one another compute the same bits: a row's logits do not depend on where it stands among 256
    or more, nor an id's among the others, and every call gives the same."""
    import torch
    from diskllm_amd import api
    x, xs, w, ws = inputs(torch, 700, 601, 520, "fp4")
    all_rows = check_product(torch, x, xs, w, ws, "fp4")
    for _ in range(5):
        assert torch.equal(api.logits_mx(x, xs, w, ws), all_rows)
    for a, b in ((0, 256), (444, 700), (17, 500)):
        assert torch.equal(api.logits_mx(x[a:b], xs[a:b], w, ws), all_rows[a:b])
    assert torch.equal(api.logits_mx(x, xs, w[89:], ws[89:]), all_rows[:, 89:])


def test_product_fp6_rows_of_odd_blocks(cuda):
    """FP6 rows that lie side by side are 8-byte aligned only."""
    import torch
    x, xs, w, ws = inputs(torch, 21, 100, 33 * 32, "fp6")
    assert x.stride(0) % 16 == 8
    check_product(torch, x, xs, w, ws, "fp6")


@pytest.mark.parametrize("rows", [2, 100, 300, 500])
@pytest.mark.parametrize("n", [96, 1024])
def test_nan_blocks_stay_in_their_rows(cuda, rows, n):
    import torch
    from diskllm_amd import api
    vocab = 300
    x, xs, w, ws = inputs(torch, rows, vocab, n, "fp4")
    xs[1, 2] = 255
    ws[299, 0] = 255
    got = api.logits_mx(x, xs, w, ws)
    bad = torch.zeros((rows, vocab), dtype=torch.bool, device="cuda")
    bad[1] = True
    bad[:, 299] = True
    assert torch.equal(got.isnan(), bad)


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("rows", [1, 16, 32, 64, 100, 200, 300, 500])
@pytest.mark.parametrize("n", [200, 1024])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e-39])
def test_product_capped_of_every_tile(cuda, fmt, rows, n, cap):
    """The cap in both formats at rows of every tile, rows of whole and of part steps."""
    import torch
    check_product(torch, *inputs(torch, rows, 301, n, fmt, seed=rows, spread=0), fmt, softcap=cap)


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("rows", [2, 16, 32, 64, 100, 200, 300, 500])
@pytest.mark.parametrize("n", [96, 1024, 1500])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_nan_blocks_of_every_tile(cuda, fmt, rows, n, cap):
    """A scale of 255 in a row's last block, in one of hidden states in the middle and in one of weights; behind a row's end
    it is none."""
    import torch
    from diskllm_amd import api
    vocab = 300
    x, xs, w, ws = inputs(torch, rows, vocab, n, fmt)
    xs[rows - 1, 1] = 255
    ws[7, -1] = 255
    ws[299, 0] = 255
    got = api.logits_mx(x, xs, w, ws, softcap=cap)
    bad = torch.zeros((rows, vocab), dtype=torch.bool, device="cuda")
    bad[rows - 1] = True
    bad[:, [7, 299]] = True
    assert torch.equal(got.isnan(), bad)
    xs[0, -1] = 255
    bad[0] = True
    assert torch.equal(api.logits_mx(x, xs, w, ws, softcap=cap).isnan(), bad)


def test_far_scales(cuda):
    """Scales at their ends: a product of a tiny and a huge block, one that underflows, one that overflows."""
    import torch
    from diskllm_amd import api
    x = torch.full((3, 32 * 4), 0.0, device="cuda")
    q, _ = api.quantize_mx(torch.ones((3, 128), device="cuda"))          # elements 4.0
    xs = torch.zeros((3, 16), dtype=torch.uint8, device="cuda")
    ws = torch.zeros((3, 16), dtype=torch.uint8, device="cuda")
    xs[0], xs[1], xs[2] = 0, 254, 100
    ws[0], ws[1], ws[2] = 254, 0, 150
    got = api.logits_mx(q, xs[:, :4], q, ws[:, :4]).cpu().double()
    want = 2048.0 * torch.exp2(xs[:, :1].cpu().double() + ws[:, 0].cpu().double()[None] - 254)
    want = torch.where(want > 3.4028235e38, float("inf"), want)
    assert ((got == want) | ((got - want).abs() <= 2.0 ** -149)).all()


@pytest.mark.parametrize("fmt", ["fp4", "fp6"])
@pytest.mark.parametrize("rows", [4, 40, 100, 200, 300])
@pytest.mark.parametrize("n", [128, 1000])
def test_tiny_products(cuda, fmt, rows, n):
    """Sums of equal products down to 2^-149, exact; below that no more than they are."""
    import torch
    from diskllm_amd import api
    vocab, blocks = 300, (n + 31) // 32
    w = torch.full((vocab, blocks * 16), 0x22, dtype=torch.uint8, device="cuda")                  # ones
    x, _ = api.quantize_mx(torch.ones((rows, blocks * 32), device="cuda"), fmt)                   # 4.0
    for total in (-126, -140, -149, -150, -153, -160, -200):
        e = 127 + (total - 2) // 2
        xs = torch.full((rows, (blocks + 15) // 16 * 16), e, dtype=torch.uint8, device="cuda")[:, :blocks]
        ws = torch.full((vocab, (blocks + 15) // 16 * 16), 254 + total - 2 - e, dtype=torch.uint8, device="cuda")[:, :blocks]
        got, want = api.logits_mx(x, xs, w, ws).double(), blocks * 32 * 2.0 ** total
        assert (got == want).all() if total >= -149 else ((got >= 0) & (got <= want + 2.0 ** -150)).all(), total


def test_offsets_past_32_bits(cuda):
    """A table of more than 2^32 bytes and logits of more than 2^32 bytes."""
    import torch
    from diskllm_amd import api
    vocab, n = 1 << 21, 4352                                    # 4.56e9 bytes of weights
    blocks = n // 32
    w = torch.full((vocab, blocks * 16), 0x22, dtype=torch.uint8, device="cuda")      # ones
    ws = torch.full((vocab, 144), 127, dtype=torch.uint8, device="cuda")[:, :blocks]
    ws[-1] = 128
    x, xs = api.quantize_mx(torch.ones((2, n), device="cuda"))
    got = api.logits_mx(x, xs, w, ws)
    assert (got[:, :-1] == n).all() and (got[:, -1] == 2 * n).all()
    e = api.dequantize_mx(w, ws, ids=torch.tensor([vocab - 1, 0], dtype=torch.int32, device="cuda"))
    assert (e[0] == 2).all() and (e[1] == 1).all()
    del w, ws, got, e
    x, xs, w, ws = inputs(torch, 300, 65, 64, "fp6")
    ld = 15_000_000                                              # 300 rows: 1.8e10 bytes
    room = torch.empty(300 * ld, device="cuda").view(300, ld)
    check_product(torch, x, xs, w, ws, "fp6", out=room[:, ld - 65:])


def test_other_stream_and_graph(cuda):
    """On a stream of its own, and captured: replays with new inputs and eager work between them."""
    import torch
    from diskllm_amd import api
    n, vocab, rows = 1000, 3000, 5
    g = torch.Generator("cuda").manual_seed(3)
    hidden = torch.randn((rows, n), device="cuda", generator=g, dtype=torch.float32).bfloat16()
    w, ws = api.quantize_mx(torch.randn((vocab, n), device="cuda", generator=g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, s = api.quantize_mx(hidden, "fp6")
        out = api.logits_mx(q, s, w, ws)
    side.synchronize()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.quantize_mx(hidden, "fp6", q=q, scale=s)
        api.logits_mx(q, s, w, ws, out=out)
    for k in range(4):
        hidden.copy_(torch.randn((rows, n), device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        again = api.logits_mx(*api.quantize_mx(hidden, "fp6"), w, ws)
        assert torch.equal(out, again)
