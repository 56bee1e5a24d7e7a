"""dlk_beam_select and dlk_beam_reorder against plain forms in 64 bits, and whole constrained searches of them."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
INF = np.float32(np.inf)


def penalised(x, ids, V, rep, freq, pres):
    """float32, the ops one after another (repetition once per occurrence, then frequency, then presence)."""
    x = x.copy()
    rep, freq, pres = np.float32(rep), np.float32(freq), np.float32(pres)
    ids = np.asarray(ids)
    ids = ids[(ids >= 0) & (ids < V)]
    for i, c in zip(*np.unique(ids, return_counts=True)):
        v = x[i]
        if rep > 1:
            for _ in range(c):
                v = np.float32(v * rep) if v < 0 else np.float32(v / rep)
        if freq != 0:
            v = np.float32(v - np.float32(freq * np.float32(c)))
        if pres != 0:
            v = np.float32(v - pres)
        x[i] = v
    return x


def allowed_bits(mask, V):
    return np.unpackbits(np.ascontiguousarray(mask).view(np.uint8), bitorder="little")[:V].astype(bool)


def select(lg, beams, n_out, scores=None, lengths=None, finished=None, hists=None, mask=None, mask_row=None, eos=-1,
           alpha=0.0, rep=1.0, freq=0.0, pres=0.0, max_history=1024):
    """The header's words in 64 bits; also the status bits."""
    rows, V = lg.shape
    groups = rows // beams
    out = dict(tokens=[], parents=[], scores=[], lengths=[], finished=[])
    status = 0
    for g in range(groups):
        cand = []
        for r in range(g * beams, (g + 1) * beams):
            cum = np.float32(0.0) if scores is None else scores[r]
            if not cum < INF:
                status |= 8
            if not (-INF < cum < INF):
                continue
            ln = 0 if lengths is None else int(lengths[r])
            if finished is not None and finished[r]:
                cand.append((float(cum) / max(ln, 1) ** alpha, r, np.inf, eos, float(cum), ln, 1))
                continue
            if hists is not None and len(hists[r]) > max_history:
                status |= 1
                continue
            x = lg[r].copy()
            if mask is not None:
                x[~allowed_bits(mask[r if mask_row is None else mask_row[r]], V)] = -np.inf
            if hists is not None:
                live = x > -np.inf
                y = penalised(np.where(live, x, np.float32(0)), hists[r], V, rep, freq, pres)
                x = np.where(live | np.isnan(x), np.where(live, y, x), -INF)
            if not (x < INF).all():
                status |= 8
                continue
            top = x.max()
            if top == -np.inf:
                continue
            x64 = x.astype(np.float64)
            with np.errstate(under="ignore"):
                z = np.log(np.exp(x64 - float(top)).sum())
            sc = float(cum) + ((x64 - float(top)) - z)
            key = sc / max(ln + 1, 1) ** alpha
            order = np.lexsort((np.arange(V), -x64, -key))
            for v in order[:n_out]:
                if x[v] > -np.inf:
                    cand.append((key[v], r, float(x[v]), int(v), sc[v], ln + 1, 1 if v == eos else 0))
        cand.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
        for j in range(n_out):
            if j < len(cand):
                _, r, _, v, sc, ln, fin = cand[j]
            else:
                r, v, sc, ln, fin = -1, -1, -np.inf, 0, 0
            for k, x in zip(out, (v, r, sc, ln, fin)):
                out[k].append(x)
    return {k: np.array(v) for k, v in out.items()}, status


def csr(hists):
    off = np.zeros(len(hists) + 1, np.int32)
    off[1:] = np.cumsum([len(h) for h in hists])
    return off, np.concatenate([np.asarray(h, np.int32) for h in hists] + [np.zeros(0, np.int32)]).astype(np.int32)


def check(torch, lg, beams, n_out, ld=None, ctx=None, **kw):
    from diskllm_amd import api
    rows, V = lg.shape
    want, status = select(lg, beams, n_out, **kw)
    room = torch.full((rows, ld or V), float("nan"), device="cuda")      # (what lies past the rows is not read)
    room[:, :V] = torch.from_numpy(lg).cuda()
    g = {k: None if kw.get(k) is None else torch.from_numpy(np.ascontiguousarray(kw[k])).cuda()
         for k in ("scores", "lengths", "finished", "mask_row")}
    if kw.get("mask") is not None:
        g["mask"] = torch.from_numpy(np.ascontiguousarray(kw["mask"]).view(np.int32)).cuda()
    if kw.get("hists") is not None:
        off, ids = csr(kw["hists"])
        g["hist_off"], g["hist_ids"] = torch.from_numpy(off).cuda(), torch.from_numpy(ids).cuda()
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = api.beam_select(room[:, :V], beams, n_out, eos_id=kw.get("eos", -1), length_penalty=kw.get("alpha", 0.0),
                          repeat_penalty=kw.get("rep", 1.0), frequency_penalty=kw.get("freq", 0.0),
                          presence_penalty=kw.get("pres", 0.0), max_history=kw.get("max_history", 0), status=st, **g)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in got.items()}
    for k in ("tokens", "parents", "lengths", "finished"):
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)
    # one rounding to float, and 64-bit sums whose exponentials are good to 1e-10
    fine = np.isfinite(want["scores"])
    np.testing.assert_array_equal(got["scores"][~fine], want["scores"][~fine].astype(np.float32))
    err = np.abs(got["scores"][fine].astype(np.float64) - want["scores"][fine])
    assert (err <= 2.0 ** -24 * np.abs(want["scores"][fine]) + 2e-10).all(), err.max()
    assert int(st.item()) == status
    return got


def logits(rng, rows, V, sd=2.5):
    return rng.normal(0, sd, (rows, V)).astype(np.float32)


@pytest.mark.parametrize("groups,beams,n_out,V", [
    (1, 1, 1, 1), (1, 1, 4, 3), (2, 3, 3, 2), (1, 4, 4, 100), (3, 2, 5, 1000), (2, 4, 4, 8191), (2, 4, 4, 8192),
    (2, 4, 8, 8193), (1, 1, 8, 32001), (5, 3, 6, 8195), (2, 16, 16, 20000), (1, 64, 64, 9001), (1, 5, 64, 16385),
    (33, 1, 2, 700), (2, 4, 4, 50257), (1, 2, 3, 151936), (1, 2, 64, 262144), (1, 64, 1, 300)])
def test_select(cuda, groups, beams, n_out, V):
    import torch
    rng = np.random.default_rng(V + beams)
    rows = groups * beams
    lg = logits(rng, rows, V)
    check(torch, lg, beams, n_out)
    check(torch, lg, beams, n_out, ld=V + 3, scores=-np.abs(rng.normal(0, 5, rows)).astype(np.float32),
          lengths=rng.integers(0, 40, rows).astype(np.int32), eos=V - 1, alpha=0.7,
          finished=(rng.random(rows) < 0.3).astype(np.uint8))


@pytest.mark.parametrize("V", [500, 8192, 30011])
@pytest.mark.parametrize("rep,freq,pres", [(1.2, 0.0, 0.0), (1.0, 0.3, 0.0), (1.0, 0.0, -2.0), (1.15, 0.25, 0.5)])
def test_select_penalties(cuda, V, rep, freq, pres):
    import torch
    rng = np.random.default_rng(V)
    lg = logits(rng, 8, V)
    best = np.argsort(-lg, axis=1)
    hists = [np.concatenate([rng.integers(-2, V + 2, 60), rng.choice(best[r, :20], 40)]) for r in range(8)]
    hists[2] = []                                                # nothing said yet
    hists[5] = [best[5, 0]] * 700 + [best[5, 1]] * 3             # one id over and over
    check(torch, lg, 4, 6, hists=hists, rep=rep, freq=freq, pres=pres,
          scores=rng.normal(-9, 2, 8).astype(np.float32))


def test_select_history_bound(cuda):
    """A row whose history passes the bound has no continuations and says so; a finished row's is not looked at."""
    import torch
    rng = np.random.default_rng(0)
    lg = logits(rng, 6, 900)
    hists = [rng.integers(0, 900, n) for n in (5, 65, 64, 65, 65, 65)]
    check(torch, lg, 3, 4, hists=hists, rep=1.3, max_history=64, eos=4, finished=np.array([0, 0, 0, 1, 1, 1], np.uint8))
    check(torch, lg, 3, 4, hists=hists, rep=1.3, max_history=64)
    long = [rng.integers(0, 900, 60000), [], [], [], [], []]
    check(torch, lg, 3, 4, hists=long, pres=0.5, freq=0.001, max_history=65535)


def mask_of(allow):
    rows, V = allow.shape
    bits = np.zeros((rows, (V + 31) // 32 * 32), np.uint8)
    bits[:, :V] = allow
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


@pytest.mark.parametrize("V", [40, 8200, 50257])
def test_select_masks(cuda, V):
    """Masks that leave a row a few ids, one or none; NaN and infinities behind a mask; masks by state."""
    import torch
    rng = np.random.default_rng(V)
    lg = logits(rng, 12, V)
    allow = rng.random((12, V)) < 0.05
    allow[1] = False
    allow[2] = False
    allow[2, V - 1] = True
    allow[4:8] = False                                           # a whole group
    allow[9, :] = True
    lg[0][~allow[0]] = np.nan
    lg[3][~allow[3]] = np.inf
    lg[8][~allow[8]] = -np.inf
    lg[10] = -np.inf
    check(torch, lg, 4, 5, mask=mask_of(allow), scores=rng.normal(-3, 1, 12).astype(np.float32))
    states = rng.integers(0, 3, 12).astype(np.int32)
    clean = logits(rng, 12, V)
    check(torch, clean, 4, 5, mask=mask_of(allow[[0, 2, 9]]), mask_row=states)
    hists = [rng.integers(0, V, 30) for _ in range(12)]
    check(torch, clean, 4, 5, mask=mask_of(allow), hists=hists, rep=1.4, freq=0.1, pres=0.2)


def test_select_not_finite(cuda):
    """Rows with NaN or +inf where it counts, scores that are not finite, logits at the ends of the range."""
    import torch
    rng = np.random.default_rng(1)
    V = 9000
    lg = logits(rng, 16, V)
    lg[0, 8999] = np.nan
    lg[1, 3] = np.inf
    lg[2] = np.finfo(np.float32).min                             # (a mask of the lowest value over everything)
    lg[3, 10:] = np.finfo(np.float32).min
    lg[4] = np.finfo(np.float32).max
    lg[5, ::2] = -np.inf
    lg[6] = 0.0
    lg[6, ::3] = -0.0                                            # equal
    lg[7, 100] = np.finfo(np.float32).max
    check(torch, lg, 4, 8)
    sc = np.array([0, -1, -np.inf, np.nan, np.inf, -3, -1e30, 5] * 2, np.float32)
    check(torch, lg, 8, 8, scores=sc)
    check(torch, lg[8:], 4, 4, scores=np.full(8, -np.inf, np.float32))


@pytest.mark.parametrize("V", [600, 8192, 24581])
@pytest.mark.parametrize("n_out", [1, 7, 64])
def test_select_equal_logits(cuda, V, n_out):
    """Runs of equal logits: the lowest rows and ids, in order."""
    import torch
    lg = np.zeros((4, V), np.float32)
    check(torch, lg, 4, n_out)
    rng = np.random.default_rng(V)
    check(torch, rng.integers(-2, 3, (4, V)).astype(np.float32), 2, n_out)
    lg = np.round(logits(rng, 4, V) * 4) / 4
    check(torch, lg, 4, n_out, scores=np.zeros(4, np.float32))
    lg[:] = np.sort(lg, axis=1)                                  # the largest side by side, at the end
    check(torch, lg, 4, n_out)
    check(torch, lg[:, ::-1].copy(), 4, n_out)


def test_select_equal_logits_many_rows(cuda):
    """Every row's first batch overflows its list: a row's entries are counted once each, whichever wave is first."""
    import torch
    from diskllm_amd import api
    lg = torch.zeros((96, 50257), device="cuda")
    for _ in range(20):
        out = api.beam_select(lg, 3, 64)
        assert (out["tokens"].view(32, 64).cpu() == torch.arange(64)).all()
        assert (out["parents"].view(32, 64).cpu() == torch.arange(0, 96, 3)[:, None]).all()


@pytest.mark.parametrize("beams,n_out,V", [(16, 16, 50257), (64, 64, 20000), (64, 64, 9001), (33, 64, 30000), (5, 11, 70000),
                                           (1, 64, 40000)])
def test_select_few_and_equal_entries(cuda, beams, n_out, V):
    """Lists of one to three entries, groups of one live row, parts of the vocabulary that are masked, scores that
    leave one row ahead, and equal logits throughout: the merges with few entries, and with too many at its bound."""
    import torch
    rng = np.random.default_rng(V + beams)
    rows = 2 * beams
    lg = logits(rng, rows, V)
    first = np.full(rows, -INF, np.float32)
    first[::beams] = 0
    check(torch, lg, beams, n_out, scores=first)
    for keep in (1, 3):
        allow = np.zeros((rows, V), bool)
        for at in range(0, V, 4096):
            allow[:, at:at + 4096 * (at % 8192 == 0):97][:, :keep] = True
        check(torch, lg, beams, n_out, mask=mask_of(allow))
    check(torch, lg, beams, n_out, mask=mask_of(np.broadcast_to(np.arange(V) % 16384 < 12288, (rows, V))))
    ahead = np.full(rows, -30, np.float32)
    ahead[beams - 1::beams] = 0
    check(torch, lg, beams, n_out, scores=ahead)
    lg[:] = 1.0
    check(torch, lg, beams, n_out)
    check(torch, lg, beams, n_out, scores=ahead)


@pytest.mark.parametrize("n_out", [1, 5, 64])
@pytest.mark.parametrize("V", [4097, 4105, 4352, 4736, 5000, 8192 + 640])
def test_select_short_ends(cuda, V, n_out):
    """Vocabularies that end in a few ids of a batch, which are a workgroup's own."""
    import torch
    rng = np.random.default_rng(V)
    check(torch, logits(rng, 8, V), 4, n_out)
    lg = logits(rng, 8, V)
    lg[:, 4096:] += 30
    check(torch, lg, 4, n_out, hists=[rng.integers(0, V, 90) for _ in range(8)], rep=1.1)


@pytest.mark.parametrize("n_out", [3, 64])
def test_select_long_slices(cuda, n_out):
    """Slices of several batches: each better than the last, or worse; equal ones; masks of all densities; histories of
    a few ids to a slice and of many in one place."""
    import torch
    rng = np.random.default_rng(n_out)
    V, rows = 70001, 64
    lg = logits(rng, rows, V)
    up = np.sort(lg, axis=1)
    check(torch, up, 64, n_out)
    check(torch, up[:, ::-1].copy(), 64, n_out)
    check(torch, np.round(lg * 2) / 2, 64, n_out)
    check(torch, np.round(up), 64, n_out)
    dense = np.concatenate([[0.0, 0.001, 1.0], np.linspace(0.02, 0.98, 61)])
    allow = rng.random((rows, V)) < dense[:, None]
    allow[5, 20000:] = False
    hidden = np.where(allow | (rng.random((rows, V)) < 0.9), lg, np.float32(np.nan))
    check(torch, hidden, 64, n_out, mask=mask_of(allow))
    best = np.argsort(-lg, axis=1)
    hists = [np.concatenate([rng.integers(-1, V + 1, 300), best[r, :40]]) for r in range(rows)]
    hists[3] = rng.integers(4096, 4300, 900)
    hists[4] = np.concatenate([np.arange(256, 512), np.arange(256, 300)])
    hists[6] = [best[6, 0]] * 64
    hists[7] = [best[7, 0]] * 65
    hists[8] = [best[8, 0]] * 60 + [best[8, 1]] * 68
    hists[12] = [best[12, 0]] * 129
    hists[13] = rng.choice(np.arange(512, 768), 120)
    kw = dict(hists=hists, rep=1.2, freq=0.2, pres=0.1)
    check(torch, lg, 64, n_out, **kw)
    check(torch, hidden, 64, n_out, mask=mask_of(allow), **kw)
    lg[9, best[9, 0]] = np.nan
    lg[10, best[10, 3]] = np.inf
    lg[11, best[11, 5]] = -np.inf
    check(torch, lg, 64, n_out, **kw)


def test_select_all_finished(cuda):
    """A group whose beams have all ended keeps them, ordered by their normalised scores."""
    import torch
    rng = np.random.default_rng(2)
    lg = np.full((8, 300), np.nan, np.float32)                   # not read
    check(torch, lg, 4, 6, finished=np.ones(8, np.uint8), eos=7, alpha=1.0, lengths=rng.integers(0, 9, 8).astype(np.int32),
          scores=rng.normal(-10, 3, 8).astype(np.float32))


def test_select_many_groups(cuda):
    """More groups than one launch's workspace holds (64 beams of 64 out)."""
    import torch
    from diskllm_amd import api
    groups, V = 63, 262145
    g = torch.Generator("cuda").manual_seed(4)
    lg = torch.randn((groups * 64, V), device="cuda", generator=g)
    sc = -torch.rand(groups * 64, device="cuda", generator=g) * 3
    out = api.beam_select(lg, 64, 64, scores=sc)
    one = [api.beam_select(lg[k * 64:(k + 1) * 64], 64, 64, scores=sc[k * 64:(k + 1) * 64]) for k in (0, 1, 35, 61, 62)]
    torch.cuda.synchronize()
    for k, o in zip((0, 1, 35, 61, 62), one):
        assert torch.equal(out["tokens"][k * 64:(k + 1) * 64], o["tokens"])
        assert torch.equal(out["parents"][k * 64:(k + 1) * 64], o["parents"] + k * 64)
        assert torch.equal(out["scores"][k * 64:(k + 1) * 64], o["scores"])


def test_select_many_rows(cuda):
    """Far more rows than workgroups that run at once, of a few ids each."""
    import torch
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(21)
    lg = torch.randn((150001, 37), device="cuda", generator=g)
    out = api.beam_select(lg, 1, 3)
    v, i = torch.sort(lg, dim=1, descending=True, stable=True)
    assert torch.equal(out["tokens"].view(-1, 3), i[:, :3].int())
    want = torch.log_softmax(lg.double(), 1).gather(1, i[:, :3]).view(-1)
    # one rounding to float, and 64-bit sums whose exponentials are good to 1e-10
    assert ((out["scores"].double() - want).abs() <= 2.0 ** -24 * want.abs() + 2e-10).all()
    assert torch.equal(out["parents"].view(-1, 3), torch.arange(150001, device="cuda").int()[:, None].expand(-1, 3))


# ---- reordering ------------------------------------------------------------------

def parents_of(rng, groups, beams, n_out, none=0.1):
    p = rng.integers(0, beams, (groups, n_out)) + np.arange(groups)[:, None] * beams
    p[rng.random((groups, n_out)) < none] = -1
    return p.reshape(-1).astype(np.int32)


@pytest.mark.parametrize("groups,beams,n_out", [(1, 1, 1), (1, 4, 4), (3, 2, 2), (2, 1, 5), (2, 8, 3), (3, 16, 16),
                                                (2, 33, 33), (1, 64, 64), (70, 3, 3)])
def test_reorder_layouts(cuda, groups, beams, n_out):
    """Caches filled in part, small rows of odd sizes at odd addresses, in place and into another buffer."""
    import torch
    from diskllm_amd import api
    rng = np.random.default_rng(groups * 100 + beams)
    p = parents_of(rng, groups, beams, n_out)
    tp = torch.from_numpy(p).cuda()
    R, N = groups * beams, groups * n_out
    g = torch.Generator("cuda").manual_seed(R)
    keep = torch.from_numpy(np.where(p < 0, 0, p)).cuda().long()
    live = torch.from_numpy(p >= 0).cuda()

    def taken(src, dst, dim, cut, length):
        """dst after the move, by indexing."""
        want = dst.clone()
        s, w = src.movedim(dim, 0), want.movedim(dim, 0)
        old = w.clone()
        new = torch.where(live.view(-1, *[1] * (s.dim() - 1)), s[keep], old)
        if cut is None:
            w.copy_(new)
        else:
            k = cut if cut < dim else cut - 1 + 1
            w.narrow(k, 0, length).copy_(new.narrow(k, 0, length))
        return want

    src = [torch.randn((3, R, 2, 10, 12), device="cuda", generator=g).to(torch.bfloat16),
           torch.randn((R, 7), device="cuda", generator=g),
           torch.randint(0, 256, (R, 40), device="cuda", generator=g, dtype=torch.uint8),
           torch.randint(0, 256, (R * 61 + 1,), device="cuda", generator=g, dtype=torch.uint8)[1:].view(R, 61)[:, :37],
           torch.randn((R,), device="cuda", generator=g),
           torch.randn((R, 2, 3000), device="cuda", generator=g).to(torch.float16),
           torch.randint(0, 256, (2, R, 9000), device="cuda", generator=g, dtype=torch.uint8),
           torch.randint(0, 9, (R, 1), device="cuda", generator=g),
           torch.randn((1, R, 1, 300, 5), device="cuda", generator=g)]
    how = [(1, 3, 7), (0, None, None), (0, None, None), (0, None, None), (0, None, None), (0, None, None),
           (1, None, None), (0, None, None), (1, 3, 299)]
    dst, want = [], []
    for s, (d, cut, length) in zip(src, how):
        shape = list(s.shape)
        shape[d] = N
        o = torch.zeros(shape, dtype=s.dtype, device="cuda")
        o.view(torch.uint8).fill_(77)
        dst.append(o)
        want.append(taken(s, o, d, cut, length))
    before = [s.clone() for s in src]
    api.beam_reorder(tp, beams, n_out, [api.beam_state(s, o, d, cut, length)
                                        for s, o, (d, cut, length) in zip(src, dst, how)])
    torch.cuda.synchronize()
    for k, (o, w, s, b) in enumerate(zip(dst, want, src, before)):
        assert torch.equal(o.view(torch.uint8), w.view(torch.uint8)), k
        assert torch.equal(s.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), k
    if beams == n_out:
        want = [taken(s, s, d, cut, length) for s, (d, cut, length) in zip(src, how)]
        api.beam_reorder(tp, beams, n_out, [api.beam_state(s, None, d, cut, length)
                                            for s, (d, cut, length) in zip(src, how)])
        torch.cuda.synchronize()
        for k, (s, w) in enumerate(zip(src, want)):
            assert torch.equal(s.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8)), k


def test_reorder_foreign_parents(cuda):
    """A parent outside the row's own group moves nothing."""
    import torch
    from diskllm_amd import api
    x = torch.arange(8, device="cuda", dtype=torch.int64).view(8, 1)
    p = torch.tensor([1, 4, -5, 2 ** 31 - 1, 7, 3, 8, 5], dtype=torch.int32, device="cuda")
    off = torch.arange(9, dtype=torch.int32, device="cuda")
    ids = torch.arange(100, 108, dtype=torch.int32, device="cuda")
    out_off, out_ids = torch.full((9,), -9, dtype=torch.int32, device="cuda"), torch.full((32,), -9, dtype=torch.int32, device="cuda")
    tok = torch.arange(8, dtype=torch.int32, device="cuda")
    api.beam_reorder(p, 4, 4, [api.beam_state(x)], api.beam_history(off, ids, tok, 4, out_off, out_ids))
    torch.cuda.synchronize()
    assert x[:, 0].tolist() == [1, 1, 2, 3, 7, 5, 6, 5]
    assert out_off.tolist() == [0, 2, 2, 2, 2, 4, 4, 4, 6]
    assert out_ids.tolist() == [101, 0, 107, 4, 105, 7] + [-9] * 26


def test_reorder_nothing(cuda):
    """No states, no groups, empty states; more states than a launch takes."""
    import torch
    from diskllm_amd import api
    p = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    api.beam_reorder(p, 2, 2)
    api.beam_reorder(torch.zeros(0, dtype=torch.int32, device="cuda"), 2, 2)
    cache = torch.randn((2, 3, 4), device="cuda")
    want = cache.clone()
    api.beam_reorder(p, 2, 2, [api.beam_state(cache, row_dim=0, length_dim=1, length=0)])
    api.beam_reorder(p, 2, 2, [api.beam_state(torch.zeros((2, 0, 3), device="cuda")), api.beam_state(torch.zeros((2, 0), device="cuda"))])
    torch.cuda.synchronize()
    assert torch.equal(cache, want)
    many = [torch.full((2, 5), float(k), device="cuda") + torch.tensor([[0.0], [0.5]], device="cuda") for k in range(21)]
    off = torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
    out_off, out_ids = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    api.beam_reorder(p, 2, 2, [api.beam_state(t) for t in many],
                     api.beam_history(off, torch.tensor([8, 9], dtype=torch.int32, device="cuda"), None, 3, out_off, out_ids))
    torch.cuda.synchronize()
    for k, t in enumerate(many):
        assert (t[0] == k + 0.5).all() and (t[1] == k).all()
    assert out_off.tolist() == [0, 0, 2] and out_ids.tolist()[:2] == [8, 9]


@pytest.mark.parametrize("groups,beams,n_out,keep", [(1, 1, 1, 1), (1, 4, 4, 5), (3, 2, 7, 40), (90, 4, 4, 300),
                                                     (5, 64, 64, 16), (384, 4, 4, 9), (385, 4, 4, 9), (5000, 1, 3, 2)])
def test_reorder_histories(cuda, groups, beams, n_out, keep):
    import torch
    from diskllm_amd import api
    rng = np.random.default_rng(groups + keep)
    R, N = groups * beams, groups * n_out
    hists = [rng.integers(0, 1000, rng.integers(0, 2 * keep + 1)) for _ in range(R)]
    if R > 1:
        hists[-1] = []
    off, ids = csr(hists)
    p = parents_of(rng, groups, beams, n_out)
    tok = rng.integers(-1, 1000, N).astype(np.int32)
    want = []
    for r in range(N):
        h = [] if p[r] < 0 else list(hists[p[r]]) + ([tok[r]] if tok[r] >= 0 else [])
        want.append(h[max(0, len(h) - keep):])
    w_off, w_ids = csr(want)
    dev = [torch.from_numpy(a).cuda() for a in (p, off, ids, tok)]
    out_off = torch.full((N + 1,), -9, dtype=torch.int32, device="cuda")
    out_ids = torch.full((N * keep,), -9, dtype=torch.int32, device="cuda")
    api.beam_reorder(dev[0], beams, n_out, history=api.beam_history(dev[1], dev[2], dev[3], keep, out_off, out_ids))
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out_off.cpu().numpy(), w_off)
    np.testing.assert_array_equal(out_ids.cpu().numpy()[:len(w_ids)], w_ids)
    assert (out_ids.cpu().numpy()[len(w_ids):] == -9).all()


def test_reorder_far_rows(cuda):
    """Offsets past 32 bits."""
    import torch
    from diskllm_amd import api
    far = (1 << 31) + 64
    big = torch.zeros(3 * far, dtype=torch.uint8, device="cuda")
    rows = torch.as_strided(big, (3, 50), (far, 1))
    x = torch.randint(0, 256, (3, 50), dtype=torch.uint8, device="cuda")
    rows.copy_(x)
    api.beam_reorder(torch.tensor([2, 0, 2], dtype=torch.int32, device="cuda"), 3, 3, [api.beam_state(rows)])
    assert torch.equal(rows, x[[2, 0, 2]])


@pytest.mark.parametrize("kind", ["bytes", "histories"])
def test_reorder_past_a_launch(cuda, kind):
    """More workgroups than a launch takes: the states, or the histories after them, go into a second one."""
    import torch
    from diskllm_amd import api
    p = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    n = (1 << 24) - (1 if kind == "histories" else 1 << 20)
    big = torch.zeros((n, 2), dtype=torch.uint8, device="cuda")            # a byte a row, n times
    big[:, 1] = 7
    small = torch.tensor([[1.0], [2.0]], device="cuda").repeat(1 << 21, 1, 1) if kind == "bytes" else torch.ones((2, 1), device="cuda")
    off = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    ids = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    out_off, out_ids = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    states = [api.beam_state(big, row_dim=1)] + ([api.beam_state(small, row_dim=1)] if kind == "bytes" else [])
    api.beam_reorder(p, 2, 2, states, api.beam_history(off, ids, None, 4, out_off, out_ids))
    torch.cuda.synchronize()
    assert (big[:, 0] == 7).all() and (big[:, 1] == 0).all()
    if kind == "bytes":
        assert (small[:, 0] == 2).all() and (small[:, 1] == 1).all()
    assert out_off.tolist() == [0, 2, 3] and out_ids.tolist() == [6, 7, 5, 0, 0, 0, 0, 0]


# ---- whole searches --------------------------------------------------------------

def text_vocab(rng, V):
    chars = np.frombuffer(b'abcdefgh0123456789{}[]"":,  ', np.uint8)
    lens = rng.integers(1, 5, V).astype(np.uint32)
    lens[V - 1] = 0
    off = np.zeros(V + 1, np.uint32)
    off[1:] = np.cumsum(lens)
    return off, chars[rng.integers(0, chars.size, int(off[-1]))]


class Search:
    """A beam search over a toy model -- the hidden state of a row is tanh(its parent's + an embedding of its token) --
    constrained by the JSON grammar, all state on the device."""

    def __init__(self, torch, groups, beams, V, n, seed, keep):
        from diskllm_amd import _lib, api
        self.t, self.api, self.L = torch, api, _lib
        self.groups, self.beams, self.V, self.n, self.keep = groups, beams, V, n, keep
        rng = np.random.default_rng(seed)
        self.off, self.bytes = text_vocab(rng, V)
        self.embed = rng.normal(0, 1, (V, n)).astype(np.float32)
        self.head = rng.normal(0, 0.3, (V, n)).astype(np.float32)
        self.first = rng.normal(0, 1, (groups, n)).astype(np.float32)
        R = groups * beams
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        z = lambda s, d: torch.zeros(s, dtype=d, device="cuda")
        self.d_off, self.d_bytes = dev(self.off.view(np.int32)), dev(self.bytes)
        self.d_embed, self.d_first = dev(self.embed), dev(self.first)
        self.w, self.ws = api.quantize_rows(dev(self.head))
        self.h = z((R, n), torch.float32)
        row = _lib.GrammarRow()
        _lib.lib().dlk_grammar_row_init(C.byref(row), _lib.GRAMMAR_JSON)
        self.fresh = dev(np.frombuffer(bytes(row) * R, np.uint8).copy().reshape(R, -1))
        self.gram = self.fresh.clone()
        self.x, self.xs = z((R, n), torch.int8), z(R, torch.float32)
        self.lg = z((R, (V + 63) // 64 * 64), torch.float32)[:, :V]
        self.mask = z((R, (V + 31) // 32), torch.int32)
        i32 = torch.int32
        self.out = [dict(tokens=z(R, i32), parents=z(R, i32), scores=z(R, torch.float32), lengths=z(R, i32),
                         finished=z(R, torch.uint8)) for _ in range(2)]
        self.hist = [(z(R + 1, i32), z(R * keep, i32)) for _ in range(2)]
        self.status = z(1, i32)
        self.reset()

    def reset(self):
        self.h.copy_(self.d_first.repeat_interleave(self.beams, 0))
        self.gram.copy_(self.fresh)
        for o in self.out:
            for k in o:
                o[k].zero_()
            o["scores"].fill_(-np.inf)
            o["scores"].view(self.groups, self.beams)[:, 0] = 0       # one beam a request to begin with
        for off, ids in self.hist:
            off.zero_()
            ids.zero_()
        self.status.zero_()

    def step(self, k):
        """Step k: from the state in slot k % 2 to the other's."""
        L, api, torch = self.L.lib(), self.api, self.t
        R, V = self.groups * self.beams, self.V
        now, new = self.out[k % 2], self.out[(k + 1) % 2]
        (off, ids), (off2, ids2) = self.hist[k % 2], self.hist[(k + 1) % 2]
        sh = api.stream_handle()
        api.quantize_rows(self.h, self.x, self.xs)
        api.logits_i8(self.x, self.xs, self.w, self.ws, softcap=8.0, out=self.lg)
        self.L.check(L.dlk_grammar_mask(self.d_off.data_ptr(), self.d_bytes.data_ptr(), V, self.gram.data_ptr(), R,
                                        V - 1, self.mask.data_ptr(), self.mask.shape[1], None, 0, None, sh), "mask")
        api.beam_select(self.lg, self.beams, self.beams, scores=now["scores"], lengths=now["lengths"],
                        finished=now["finished"], hist_off=off, hist_ids=ids, mask=self.mask, eos_id=V - 1,
                        length_penalty=0.6, repeat_penalty=1.1, presence_penalty=0.3, max_history=self.keep,
                        out=new, status=self.status)
        api.beam_reorder(new["parents"], self.beams, self.beams, [api.beam_state(self.h), api.beam_state(self.gram)],
                         api.beam_history(off, ids, new["tokens"], self.keep, off2, ids2))
        self.L.check(L.dlk_grammar_advance(self.d_off.data_ptr(), self.d_bytes.data_ptr(), V, self.gram.data_ptr(),
                                           new["tokens"].data_ptr(), R, V - 1, sh), "advance")
        self.h.add_(self.d_embed[new["tokens"].clamp(min=0).long()]).tanh_()


@pytest.mark.parametrize("groups,beams,V,n", [(1, 4, 700, 64), (3, 3, 2500, 100), (2, 8, 9000, 33)])
def test_search(cuda, groups, beams, V, n):
    """Every step of a search against the plain forms: the logits the step selected from, the grammar masks by the
    validators' host form, the histories, the states."""
    import torch
    from test_gpu_logits_i8 import product, quantized
    s = Search(torch, groups, beams, V, n, seed=V, keep=6)
    R = groups * beams
    texts, hists = [b""] * R, [[] for _ in range(R)]
    h = np.repeat(s.first, beams, 0)
    row = s.L.GrammarRow
    mode_rows = []
    for _ in range(R):
        r = row()
        s.L.lib().dlk_grammar_row_init(C.byref(r), s.L.GRAMMAR_JSON)
        mode_rows.append(r)
    qw, sw = quantized(s.head)
    np.testing.assert_array_equal(s.w.cpu().numpy(), qw)
    live = 0
    for k in range(9):
        now = {key: v.cpu().numpy().copy() for key, v in s.out[k % 2].items()}
        s.step(k)
        torch.cuda.synchronize()
        lg = s.lg.cpu().numpy()
        qx, sx = quantized(h)
        want = 8.0 * np.tanh(product(qx, sx, qw, sw) / 8.0)
        assert np.abs(lg - want).max() <= 8.0 * 2.0 ** -20              # (16 half-steps of the cap)
        got = {key: v.cpu().numpy() for key, v in s.out[(k + 1) % 2].items()}
        exp, status = select(lg, beams, beams, scores=now["scores"], lengths=now["lengths"], finished=now["finished"],
                             hists=hists, mask=s.mask.cpu().numpy().view(np.uint32), eos=V - 1, alpha=0.6, rep=1.1,
                             pres=0.3)
        for key in ("tokens", "parents", "lengths", "finished"):
            np.testing.assert_array_equal(got[key], exp[key], err_msg=f"step {k} {key}")
        assert status == 0 and int(s.status.item()) == 0
        # the states follow
        p, tok = exp["parents"], exp["tokens"]
        old = (hists, [bytes(r) for r in mode_rows], h)
        hists = [[] if p[r] < 0 else (list(old[0][p[r]]) + [tok[r]])[-6:] for r in range(R)]
        fed = []
        for r in range(R):
            st = row.from_buffer_copy(old[1][p[r] if p[r] >= 0 else r])
            if tok[r] >= 0 and tok[r] != V - 1:
                piece = bytes(s.bytes[s.off[tok[r]]:s.off[tok[r] + 1]])
                s.L.lib().dlk_grammar_row_feed(C.byref(st), piece, len(piece))
            fed.append(st)
        mode_rows = fed
        np.testing.assert_array_equal(s.gram.cpu().numpy(), np.frombuffer(b"".join(bytes(r) for r in fed), np.uint8).reshape(R, -1))
        off, ids = (a.cpu().numpy() for a in s.hist[(k + 1) % 2])
        for r in range(R):
            assert ids[off[r]:off[r + 1]].tolist() == hists[r]
        base = np.stack([old[2][p[r] if p[r] >= 0 else r] for r in range(R)])
        h = s.h.cpu().numpy()
        near = np.tanh(base.astype(np.float64) + s.embed[np.maximum(tok, 0)])
        assert np.abs(h - near).max() < 1e-6
        live = max(live, int((tok >= 0).sum()))
    assert live == R


def test_search_replayed(cuda):
    """Two steps captured in a graph (from one slot to the other and back), replayed with eager work in between, give
    what eager steps give."""
    import torch
    s = Search(torch, 2, 4, 1500, 64, seed=9, keep=16)
    for k in range(8):
        s.step(k)
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in s.out[0].items()}
    gram, hid, hist = s.gram.clone(), s.h.clone(), [t.clone() for t in s.hist[0]]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        s.reset()
        s.step(0)
        s.step(1)                                                # (this stream's workspace)
        st.synchronize()
        s.reset()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        s.step(0)
        s.step(1)
    for _ in range(3):
        s.reset()
        for _ in range(4):
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            torch.zeros(1000, device="cuda").add_(1).sum().item()
        for k in want:
            assert torch.equal(s.out[0][k], want[k]), k
        assert torch.equal(s.gram, gram) and torch.equal(s.h, hid)
        assert torch.equal(s.hist[0][0], hist[0])
        n = int(hist[0][-1])
        assert torch.equal(s.hist[0][1][:n], hist[1][:n])
    del g
    from diskllm_amd import _lib
    _lib.check(_lib.lib().dlk_release_stream(st.cuda_stream), "dlk_release_stream")


def test_capture_without_workspace_is_refused(cuda):
    import torch
    from diskllm_amd import _lib, api
    lg = torch.randn((4, 300), device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    _lib.check(_lib.lib().dlk_release_stream(st.cuda_stream), "dlk_release_stream")
    g = torch.cuda.CUDAGraph()
    out = api.beam_select(lg, 4, 4)
    with torch.cuda.graph(g, stream=st):
        lg.mul_(1.0)
        with pytest.raises(RuntimeError):
            api.beam_select(lg, 4, 4, out=out)
    g.replay()
    torch.cuda.synchronize()


def test_calls_of_all_sizes_on_one_stream(cuda):
    """Calls that share a workspace one after another, each smaller or larger than the last, and dlk_sample between
    them; the same into a graph, replayed with such calls in between."""
    import torch
    from diskllm_amd import _lib, api
    from diskllm_amd import workloads as W
    g = torch.Generator("cuda").manual_seed(12)
    sizes = [(4, 4, 4, 32000), (64, 8, 16, 50257), (2, 1, 64, 700), (16, 16, 3, 9001), (192, 64, 64, 30000)]
    lg = [torch.randn((r, v), device="cuda", generator=g) for r, _, _, v in sizes]
    db = api.to_device(W.c3(rows=4, vocab=4099))
    api.sample(db)
    ids = db.out_ids.clone()
    alone = []
    for x, (_, b, n, _) in zip(lg, sizes):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            st.wait_stream(torch.cuda.default_stream())
            alone.append(api.beam_select(x, b, n))
            st.synchronize()
        _lib.check(_lib.lib().dlk_release_stream(st.cuda_stream), "dlk_release_stream")
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for k in (0, 1, 2, 3, 4, 2, 0, 4, 1):
            got = api.beam_select(lg[k], *sizes[k][1:3])
            db.reset_rng()
            api.sample(db)
            assert torch.equal(db.out_ids, ids)
            for name in got:
                assert torch.equal(got[name], alone[k][name]), (k, name)
    st.synchronize()
    outs = [{k: torch.zeros_like(v) for k, v in a.items()} for a in alone]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        for x, (_, b, n, _), o in zip(lg, sizes, outs):
            api.beam_select(x, b, n, out=o)
    for k in (4, 0, 2):
        for o in outs:
            for v in o.values():
                v.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            got = api.beam_select(lg[k], *sizes[k][1:3])
            graph.replay()
        torch.cuda.synchronize()
        for a, o in zip(alone + [alone[k]], outs + [got]):
            for name in a:
                assert torch.equal(a[name], o[name]), name
    del graph
    _lib.check(_lib.lib().dlk_release_stream(st.cuda_stream), "dlk_release_stream")


def test_streams_at_once(cuda):
    """Searches on three streams at once, each with its own workspace."""
    import torch
    from diskllm_amd import _lib, api
    g = torch.Generator("cuda").manual_seed(8)
    lg = [torch.randn((32, 60000), device="cuda", generator=g) for _ in range(3)]
    want = [api.beam_select(x, 4, 8) for x in lg]
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [{k: torch.zeros_like(v) for k, v in w.items()} for w in want]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, st, o in zip(lg, streams, outs):
            with torch.cuda.stream(st):
                api.beam_select(x, 4, 8, out=o)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for k in w:
            assert torch.equal(w[k], o[k]), k
    for st in streams:
        _lib.check(_lib.lib().dlk_release_stream(st.cuda_stream), "dlk_release_stream")


def test_outputs_on_a_given_stream(cuda):
    """A stream by its handle while the current one still has work for blocks of the outputs' sizes, just freed: the
    outputs are other memory.  The same from a side stream onto the default one."""
    import torch
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(2)
    h = torch.randn((40, 320), device="cuda", generator=g)
    w, ws = api.quantize_rows(torch.randn((1000, 320), device="cuda", generator=g))
    want_q, want_s = api.quantize_rows(h)
    want_l = api.logits_i8(want_q, want_s, w, ws)
    want_b = api.beam_select(want_l, 4, 4)
    busy = torch.empty(1 << 28, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for current, other in ((torch.cuda.default_stream(), side.cuda_stream), (side, 0)):
        with torch.cuda.stream(current):
            held = [torch.empty_like(t) for t in (want_q, want_s, want_l, *want_b.values())]
            held.append(torch.empty((3, 40), dtype=torch.int32, device="cuda"))
            for _ in range(20):
                busy.fill_(1.0)
            for t in held:
                t.fill_(3)
            del held, t
            q, s = api.quantize_rows(h, stream=other)
            logits = api.logits_i8(q, s, w, ws, stream=other)
            out = api.beam_select(logits, 4, 4, stream=other)
        torch.cuda.synchronize()
        assert torch.equal(q, want_q) and torch.equal(s, want_s) and torch.equal(logits, want_l)
        assert all(torch.equal(out[k], want_b[k]) for k in out)


@pytest.mark.parametrize("V,shape", [(2, "pair"), (40, "pair"), (5000, "spread"), (20000, "rising"), (20000, "falling"),
                                     (100000, "rising"), (50257, "level")])
def test_select_orders_near_rows(cuda, V, shape):
    """A row of one continuation beside a row of many, their best scores a few times the header's bound apart, in
    either direction.  The gap is set by one logit of the second row and is known from sums in 64 bits."""
    import torch
    from diskllm_amd import api
    rng = np.random.default_rng(V)
    if shape == "pair":
        base, grid, at = np.zeros(1, np.float32), -rng.uniform(0.05, 3.0, 1 << 22).astype(np.float32), 1
    else:
        base = {"spread": lambda: rng.normal(0, 2.5, V - 1), "rising": lambda: np.linspace(-20, 0, V - 1),
                "falling": lambda: np.linspace(0, -20, V - 1), "level": lambda: np.full(V - 1, -1e-3)}[shape]().astype(np.float32)
        base -= base.max()
        base[0 if shape == "falling" else -1] = 0.0
        grid, at = -rng.uniform(0.05, 3.0, 1 << 22).astype(np.float32), V // 2
    import math
    rest = math.fsum(np.exp(base.astype(np.float64))) - 1.0
    best = -np.log1p(rest + np.exp(grid.astype(np.float64)))          # the second row's best score, for each value
    other = best.astype(np.float32)                                   # the first row's, a float beside it
    gap = best - other.astype(np.float64)
    size = np.abs(best)
    # past the bound, and past what this sum in 64 bits may be off by
    room = 2.0 ** -42 + 2.0 ** -50 * size
    pick = np.flatnonzero((np.abs(gap) > 1.25 * room) & (np.abs(gap) < 1.25 * room + 4e-12))
    assert len(pick) >= 24
    pick = np.concatenate([pick[gap[pick] > 0][:64], pick[gap[pick] < 0][:64]])
    groups = len(pick)
    lg = np.full((2 * groups, V), -np.inf, np.float32)
    lg[0::2, 0] = 0.0
    lg[1::2, :at] = base[:at]
    lg[1::2, at] = grid[pick]
    if V > at + 1:
        lg[1::2, at + 1:at + 1 + len(base) - at] = base[at:]
    top = int(lg[1].argmax())
    scores = np.zeros(2 * groups, np.float32)
    scores[0::2] = other[pick]
    got = api.beam_select(torch.from_numpy(lg).cuda(), 2, 2, scores=torch.from_numpy(scores).cuda())
    torch.cuda.synchronize()
    parents, tokens = got["parents"].cpu().numpy().reshape(groups, 2), got["tokens"].cpu().numpy().reshape(groups, 2)
    second_first = gap[pick] > 0
    np.testing.assert_array_equal(parents[:, 0] & 1, second_first)
    np.testing.assert_array_equal(tokens[:, 0], np.where(second_first, top, 0))
    assert second_first.any() and not second_first.all()


def late(rng, groups, beams, score):
    """Scores of beams late in a long search: far from 0 and near one another."""
    return (score - rng.uniform(0, 0.6, (groups, beams)).cumsum(1)).astype(np.float32).reshape(-1)


@pytest.mark.parametrize("score", [-600.0, -1200.0, -4000.0, -1e6, -1e30])
@pytest.mark.parametrize("groups,beams,n_out,V", [(2, 4, 4, 9000), (2, 16, 16, 50257), (2, 8, 16, 50257), (1, 16, 32, 128256),
                                                  (1, 64, 64, 20000), (3, 1, 64, 151936)])
def test_select_far_scores(cuda, groups, beams, n_out, V, score):
    import torch
    rng = np.random.default_rng(V + beams)
    lg = logits(rng, groups * beams, V)
    sc = late(rng, groups, beams, score)
    if score > -1e5:
        check(torch, lg, beams, n_out, scores=sc)
        check(torch, lg, beams, n_out, scores=sc, lengths=rng.integers(300, 900, groups * beams).astype(np.int32), alpha=0.7,
              eos=7, finished=(rng.random(groups * beams) < 0.3).astype(np.uint8))
        check(torch, lg + np.float32(1000), beams, n_out, scores=sc)
    else:
        # (a score's 64 bits no longer tell all entries apart: equal ones by the lower row, the larger logit, the lower id)
        check(torch, lg, beams, n_out, scores=sc)


@pytest.mark.parametrize("groups,beams,n_out,V", [(8, 16, 16, 50257), (8, 8, 16, 50257), (16, 16, 32, 128256)])
def test_select_far_scores_cost_no_more(cuda, groups, beams, n_out, V):
    """How far the scores are from 0 does not decide how the lists are merged: taken one by one, 16 continuations cost
    half of the whole call again."""
    import torch
    rng = np.random.default_rng(4)
    assert_costs_alike(torch, groups, beams, n_out, V, *(late(rng, groups, beams, s) for s in (-2.0, -2500.0)))


def assert_costs_alike(torch, groups, beams, n_out, V, few, many):
    """A selection with the scores `many` takes no more than a quarter longer than with `few`, by their best of 15 turns."""
    from diskllm_amd import api
    g = torch.Generator("cuda").manual_seed(3)
    lg = torch.randn((groups * beams, V), device="cuda", generator=g) * 2.5
    scores = [torch.from_numpy(s).cuda() for s in (few, many)]
    out = api.beam_select(lg, beams, n_out, scores=scores[0])
    best = [1e9, 1e9]
    for _ in range(15):
        for k, sc in enumerate(scores):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            api.beam_select(lg, beams, n_out, scores=sc, out=out)
            start.record()
            for _ in range(20):
                api.beam_select(lg, beams, n_out, scores=sc, out=out)
            end.record()
            end.synchronize()
            best[k] = min(best[k], start.elapsed_time(end))
    assert best[1] < 1.25 * best[0], best


@pytest.mark.parametrize("groups,beams,V", [(16, 2, 151936), (16, 4, 151936)])
def test_select_near_beams_cost_no_more(cuda, groups, beams, V):
    """64 continuations that may come from any beam of a group, beside those of one beam alone."""
    import torch
    few = np.tile(np.where(np.arange(beams) == 0, -5.0, -5000.0), groups).astype(np.float32)
    assert_costs_alike(torch, groups, beams, 64, V, few, late(np.random.default_rng(4), groups, beams, -5.0))


def test_select_scores_beside_zero(cuda):
    """Scores so small, on both sides of 0, that their distances over the lengths are no floats: still in order."""
    import torch
    rng = np.random.default_rng(8)
    rows = 64
    lg = np.full((rows, 3), -np.inf, np.float32)
    lg[:, 1] = rng.normal(0, 3, rows)                  # one continuation a row, its log-softmax 0
    for sign in (1.0, -1.0, 0.0):
        s = (10.0 ** rng.uniform(-44, -36, rows) * (sign or rng.choice([-1, 1], rows))).astype(np.float32)
        s = np.unique(s)
        s = rng.permutation(s)[:len(s) // 16 * 16]
        n = len(s)
        check(torch, lg[:n], 16, 5, scores=s, lengths=np.full(n, 500, np.int32), alpha=16.0)
        check(torch, lg[:n], 16, 16, scores=s, lengths=np.full(n, 500, np.int32), alpha=16.0)
        check(torch, lg[:n], 16, 5, scores=s)
