"""dlk_quantize_rows and dlk_logits_i8 against plain forms in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                        # half a step of float32, relative


def quantized(x):
    """(q, scale) of float32 rows as the header says, the rounding of the quotient decided exactly: scale * (n + 1/2)
    has at most 33 significant bits, and its difference from an x next to it fits 64-bit floats too."""
    x64 = x.astype(np.float64)
    amax = np.abs(x64).max(1)
    bad = ~np.isfinite(amax) | np.isnan(x64).any(1)
    with np.errstate(all="ignore"):
        scale = (amax / 127.0).astype(np.float32)
        t = x64 / scale[:, None].astype(np.float64)
        n = np.floor(t)
        d = x64 - (n + 0.5) * scale[:, None].astype(np.float64)
        q = np.where(d > 0, n + 1, np.where(d < 0, n, 2 * np.floor((n + 1) / 2)))
    q = np.where(scale[:, None] > 0, q, 0)
    q[bad] = 0
    scale[bad] = np.nan
    return np.clip(q, -127, 127).astype(np.int8), scale


def check_quantized(torch, x, **kw):
    from diskllm_amd import api
    q, s = api.quantize_rows(x, **kw)
    torch.cuda.synchronize()
    want_q, want_s = quantized(x.float().cpu().numpy())
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    return q, s


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,n,pad", [(1, 1, 0), (1, 7, 0), (3, 8, 3), (5, 511, 0), (130, 1024, 5), (2, 1025, 0),
                                        (1, 4096, 0), (33, 8192, 8), (4, 8193, 1), (3, 20011, 0)])
def test_quantize(cuda, dtype, rows, n, pad):
    import torch
    g = torch.Generator("cuda").manual_seed(rows * 1000 + n)
    x = torch.randn((rows, n + pad), device="cuda", generator=g) * 3
    check_quantized(torch, x.to(getattr(torch, dtype))[:, :n])


def test_quantize_special_rows(cuda):
    """Zeros, halves that go to the even value, NaN, infinities, the smallest and largest magnitudes."""
    import torch
    n = 200
    x = np.zeros((12, n), np.float32)
    x[1] = np.arange(n) % 128 + 0.5
    x[1, 0] = 127.0                                              # scale 1: every quotient is a half
    x[2] = -(np.arange(n) % 127) - 0.5
    x[2, 5] = 127.0
    x[3, 7] = np.nan
    x[4, 150] = np.inf
    x[5, 199] = -np.inf
    x[6] = np.float32(1e-45) * np.arange(n)                      # subnormal: the scale loses nearly all its bits
    x[7] = np.float32(1e-38) * np.linspace(-1, 1, n)
    x[8] = np.float32(3e38) * np.linspace(-1, 1, n)
    x[9, 3] = np.float32(1e-45)                                  # scale rounds to 0
    x[10] = -0.0
    x[11] = np.float32(1.9e-30) * np.linspace(-127, 127, n)      # next to where the quotient's form changes
    q, s = check_quantized(torch, torch.from_numpy(x).cuda())
    assert torch.isnan(s[3:6]).all() and s[0] == 0 and s[9] == 0


def test_quantize_into_strided(cuda):
    """Into rows of any stride and alignment; what lies between the rows is left."""
    import torch
    x = torch.randn((9, 100), device="cuda")
    room = torch.full((9 * 131 + 1,), 77, dtype=torch.int8, device="cuda")
    q = room[1:].view(9, 131)[:, :100]
    scale = torch.zeros(11, device="cuda")
    check_quantized(torch, x, q=q, scale=scale[:9])
    assert (room[1:].view(9, 131)[:, 100:] == 77).all() and room[0] == 77 and (scale[9:] == 0).all()


def product(x, xs, w, ws):
    """In 64 bits: the sums are whole numbers below 2^53."""
    return (x.astype(np.float64) @ w.astype(np.float64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)


def int8(rng, rows, n, ld, offset):
    buf = rng.integers(-128, 128, rows * ld + 16 + offset, dtype=np.int8)
    return buf, np.lib.stride_tricks.as_strided(buf[offset:], (rows, n), (ld, 1))


def on_gpu(torch, buf, rows, n, ld, offset):
    """The rows in a buffer that ends with the last row: a read past it is a read past the tensor."""
    t = torch.from_numpy(buf[:offset + (rows - 1) * ld + n].copy()).cuda()
    return torch.as_strided(t, (rows, n), (ld, 1), offset)


SHAPES = [(1, 1, 1), (1, 64, 64), (2, 17, 5), (3, 100, 16), (5, 33, 15), (16, 257, 127), (17, 300, 512), (31, 129, 640),
          (33, 1000, 2047), (64, 511, 1024), (65, 200, 130), (100, 333, 259), (128, 130, 384), (129, 257, 1000),
          (255, 300, 256), (257, 513, 320), (300, 700, 77), (513, 100, 200)]


@pytest.mark.parametrize("rows,V,n", SHAPES)
@pytest.mark.parametrize("layout", ["padded", "packed", "odd"])
def test_logits(cuda, rows, V, n, layout):
    import torch
    from diskllm_amd import api
    rng = np.random.default_rng(rows * 7919 + V * 31 + n)
    ld, off = {"padded": ((n + 15) // 16 * 16, 0), "packed": (n, 0), "odd": (n + 3, 1)}[layout]
    xb, x = int8(rng, rows, n, ld, off)
    wb, w = int8(rng, V, n, ld, off)
    xs = rng.uniform(0.001, 0.1, rows).astype(np.float32)
    ws = rng.uniform(0.0001, 0.01, V).astype(np.float32)
    ldo = V if layout == "packed" else V + 5
    room = torch.full((rows, ldo), 123.0, device="cuda")
    out = room[:, :V]
    api.logits_i8(on_gpu(torch, xb, rows, n, ld, off), torch.from_numpy(xs).cuda(),
                  on_gpu(torch, wb, V, n, ld, off), torch.from_numpy(ws).cuda(), out=out)
    torch.cuda.synchronize()
    want = product(x, xs, w, ws)
    # the sum's rounding, then one for each scale: three halves of a step
    err = np.abs(out.cpu().numpy().astype(np.float64) - want)
    assert (err <= 3.01 * U * np.abs(want)).all(), (err / np.maximum(np.abs(want), 1e-30)).max() / U
    assert (room[:, V:] == 123.0).all()


@pytest.mark.parametrize("n", [5, 16, 100, 513, 1025, 2047])
@pytest.mark.parametrize("rows,V", [(1, 300), (1, 1), (40, 1)])
def test_logits_single_rows(cuda, rows, V, n):
    """One row of x or of w whose stride is no multiple of 16, in a buffer that ends with it."""
    import torch
    from diskllm_amd import api
    rng = np.random.default_rng(n)
    pad = (n + 15) // 16 * 16
    ldx, ldw = n if rows == 1 else pad, n if V == 1 else pad
    xb, x = int8(rng, rows, n, ldx, 0)
    wb, w = int8(rng, V, n, ldw, 0)
    out = api.logits_i8(on_gpu(torch, xb, rows, n, ldx, 0), torch.ones(rows, device="cuda"),
                        on_gpu(torch, wb, V, n, ldw, 0), torch.ones(V, device="cuda"))
    np.testing.assert_array_equal(out.cpu().numpy(), product(x, np.ones(rows), w, np.ones(V)).astype(np.float32))


def test_logits_extreme_sums(cuda):
    """-128 * -128 at the largest n: the sum's 32 bits are just enough."""
    import torch
    from diskllm_amd import api
    n = 131071
    x = torch.full((1, n), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, n), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, 1:] = 0
    out = api.logits_i8(x, torch.ones(1, device="cuda"), w, torch.ones(3, device="cuda"))
    assert out[0].tolist() == [float(np.float32(n * 16384)), float(np.float32(-n * 128 * 127)), 16384.0]


@pytest.mark.parametrize("rows,V,n", [(1, 1003, 64), (20, 2000, 96), (130, 515, 128), (400, 260, 64)])
@pytest.mark.parametrize("cap", [30.0, 5.0, 0.01, 1e-30, 1e30])
def test_logits_softcap(cuda, rows, V, n, cap):
    import torch
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(V)
    x = torch.randint(-127, 128, (rows, n), device="cuda", generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (V, n), device="cuda", generator=g, dtype=torch.int8)
    w[3] = 0
    xs, ws = torch.rand(rows, device="cuda", generator=g) * 0.02, torch.rand(V, device="cuda", generator=g) * 0.1
    xs *= torch.exp(torch.randn(rows, device="cuda", generator=g))
    ws *= torch.exp(torch.randn(V, device="cuda", generator=g) * 4)             # quotients from 1e-6 to far past 1
    xs[0], ws[7] = float("nan"), float("inf")                    # (rows that could not be quantised)
    plain = api.logits_i8(x, xs, w, ws).double()
    got = api.logits_i8(x, xs, w, ws, softcap=cap).double()
    torch.cuda.synchronize()
    c = float(np.float32(cap))
    want = c * torch.tanh(plain / c)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    err = ((got - want).abs() / want.abs().clamp(min=1e-37)).nan_to_num()
    # two roundings of the quotient, the series' or the exponential's (4.5 half-steps where it is worst), of 1 + e, its
    # reciprocal and the products, and the product with the cap: below 16 half-steps
    assert float(err.max()) <= 16 * U, float(err.max()) / U


@pytest.mark.parametrize("rows", [1, 20, 130, 400])
@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("cap", [1e-45, 1e-40, 2.9387e-39, 2.0 ** -128, 3e-39, 1e-38, 3.4e38])
def test_logits_softcap_extreme(cuda, rows, layout, cap):
    """Caps whose reciprocal is no float, next to those that have one, and the largest; what lies past a row is left."""
    import torch
    from diskllm_amd import api
    V, n = 261, 65
    g = torch.Generator("cuda").manual_seed(rows)
    ld = n if layout == "packed" else 80
    x = torch.randint(-127, 128, (rows, ld), device="cuda", generator=g, dtype=torch.int8)[:, :n]
    w = torch.randint(-127, 128, (V, ld), device="cuda", generator=g, dtype=torch.int8)[:, :n]
    w[3] = 0
    c = float(np.float32(cap))
    # sums of some 5e4 by sqrt(c) / 3e2 twice: quotients about 1/2; some rows and ids far below and above
    xs = torch.full((rows,), float(np.sqrt(c) / 300), device="cuda") * torch.exp(torch.randn(rows, device="cuda", generator=g))
    ws = torch.full((V,), float(np.sqrt(c) / 300), device="cuda") * torch.exp(torch.randn(V, device="cuda", generator=g) * 4)
    plain = api.logits_i8(x, xs, w, ws).double()
    room = torch.full((rows, V + 3), 7.0, device="cuda")
    api.logits_i8(x, xs, w, ws, softcap=cap, out=room[:, :V])
    torch.cuda.synchronize()
    got = room[:, :V].double()
    want = c * torch.tanh(plain / c)
    # 16 half-steps as above; the reciprocal of a cap past 2^126 is off by up to 4; a subnormal result's own rounding,
    # and the quotient's where that is subnormal
    room_for = (16 + (4 if cap > 2.0 ** 126 else 0)) * U * want.abs() + 2.0 ** -149 + 2.0 ** -148 * c
    assert ((got - want).abs() <= room_for).all(), float(((got - want).abs() - room_for).max())
    assert (room[:, V:] == 7.0).all()


def test_hidden_states_to_logits(cuda):
    """The two calls as a decode step makes them; a token whose hidden state is not finite has NaN logits and leaves
    the others alone."""
    import torch
    from diskllm_amd import api
    rng = np.random.default_rng(3)
    h = torch.from_numpy(rng.normal(0, 1, (6, 200)).astype(np.float32)).cuda().to(torch.bfloat16)
    W = torch.from_numpy(rng.normal(0, 0.1, (999, 200)).astype(np.float32)).cuda()
    h[2, 9] = float("inf")
    x, xs = api.quantize_rows(h)
    w, ws = api.quantize_rows(W)
    out = api.logits_i8(x, xs, w, ws)
    torch.cuda.synchronize()
    (qx, sx), (qw, sw) = quantized(h.float().cpu().numpy()), quantized(W.cpu().numpy())
    want = product(qx, sx, qw, sw)
    got = out.cpu().numpy()
    assert np.isnan(got[2]).all()
    fine = [0, 1, 3, 4, 5]
    assert (np.abs(got[fine] - want[fine]) <= 3.01 * U * np.abs(want[fine])).all()
    # next to the unquantised product: each value is off by at most half its scale
    full = h.float().cpu().numpy().astype(np.float64) @ W.cpu().numpy().astype(np.float64).T
    x64, w64 = np.abs(h.float().cpu().numpy().astype(np.float64)), np.abs(W.cpu().numpy().astype(np.float64))
    for r in fine:
        room = 0.5 * sx[r] * w64.sum(1) + 0.5 * sw * x64[r].sum() + 0.25 * sx[r] * sw * 200
        assert (np.abs(got[r] - full[r]) <= room * 1.001).all()


def test_replayed_graph(cuda):
    """Captured and replayed with other inputs in the same buffers, eager work in between."""
    import torch
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(5)
    h = torch.randn((12, 300), device="cuda", generator=g)
    W = torch.randn((700, 300), device="cuda", generator=g)
    w, ws = api.quantize_rows(W)
    x, xs = api.quantize_rows(h)
    out = api.logits_i8(x, xs, w, ws, softcap=20.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.quantize_rows(h, x, xs)
        api.logits_i8(x, xs, w, ws, softcap=20.0, out=out)
    for k in range(3):
        h.copy_(torch.randn((12, 300), device="cuda", generator=g) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        x2, xs2 = api.quantize_rows(h)
        want = api.logits_i8(x2, xs2, w, ws, softcap=20.0)
        torch.cuda.synchronize()
        assert torch.equal(x, x2) and torch.equal(xs, xs2) and torch.equal(out, want)


def test_rows_far_apart(cuda):
    """Rows whose offsets pass 32 bits, in and out."""
    import torch
    from diskllm_amd import api
    far = (1 << 31) + 4096
    n, V = 96, 40
    big = torch.zeros(2 * far, dtype=torch.int8, device="cuda")
    w = torch.as_strided(big, (2, n), (far, 1))
    g = torch.Generator("cuda").manual_seed(1)
    w.copy_(torch.randint(-127, 128, (2, n), device="cuda", generator=g, dtype=torch.int8))
    x = torch.randint(-127, 128, (V, n), device="cuda", generator=g, dtype=torch.int8)
    one, two = torch.ones(V, device="cuda"), torch.ones(2, device="cuda")
    want = (x.double() @ w.double().t()).float()
    assert torch.equal(api.logits_i8(x, one, w, two), want)              # far rows of weights
    assert torch.equal(api.logits_i8(w, two, x, one), want.t())          # far rows of x
    q = torch.as_strided(big, (2, n), (far, 1))
    h = torch.randn((2, n), device="cuda", generator=g)
    check_quantized(torch, h, q=q)
    del big, w, q
    out = torch.as_strided(torch.zeros(far + V, device="cuda"), (2, V), (far, 1))
    w2 = torch.randint(-127, 128, (2, n), device="cuda", generator=g, dtype=torch.int8)
    want = (w2.double() @ x.double().t()).float()
    assert torch.equal(api.logits_i8(w2, two, x, one, out=out), want)


@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 384, 385, 512, 520, 700])
@pytest.mark.parametrize("n", [64, 512, 1000, 1536])
@pytest.mark.parametrize("packed", [False, True])
def test_logits_tiles(cuda, rows, n, packed):
    """Every tile, full and partly filled, one stage, several, and a shorter last one; the sums are exact."""
    import torch
    from diskllm_amd import api
    V = 777
    g = torch.Generator("cuda").manual_seed(rows + n)
    ld = n + 1 if packed else (n + 15) // 16 * 16
    x = torch.randint(-128, 128, (rows, ld), device="cuda", generator=g, dtype=torch.int8)[:, :n]
    w = torch.randint(-128, 128, (V, ld), device="cuda", generator=g, dtype=torch.int8)[:, :n]
    one, each = torch.ones(rows, device="cuda"), torch.ones(V, device="cuda")
    out = api.logits_i8(x, one, w, each)
    want = (x.double() @ w.double().t()).float()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
