"""What dlk_quantize_mx, dlk_dequantize_mx, dlk_logits_mx, dlk_token_logprobs and dlk_token_logprobs_grad refuse, before any
device work: through the C entry points with addresses that are never read, and through the Python functions with CPU
tensors."""
import ctypes as C

import pytest
import torch

from diskllm_amd import _lib, api

A = 1 << 20                       # some 16-byte aligned address
INV, UNS, OK = _lib.DLK_ERR_INVALID, _lib.DLK_ERR_UNSUPPORTED, _lib.DLK_OK
FP4, FP6 = _lib.MX_FP4, _lib.MX_FP6


def call(fn, base, **kw):
    """fn with base's arguments (in order), some of them changed."""
    a = dict(base)
    assert set(kw) <= set(a)
    a.update(kw)
    return fn(*a.values())


QUANT = dict(x=A, dtype=_lib.BF16, ldx=64, rows=2, n=64, format=FP4, q=A, ldq=32, scale=A, lds=2, stream=None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), INV), (dict(q=None), INV), (dict(scale=None), INV), (dict(rows=-1), INV), (dict(n=0), INV),
    (dict(ldx=63), INV), (dict(ldq=24), INV), (dict(format=FP6, ldq=40), INV), (dict(lds=1), INV), (dict(dtype=3), INV),
    (dict(format=2), INV), (dict(format=-1), INV), (dict(x=A + 1), INV), (dict(x=A + 2, dtype=_lib.F32), INV),
    (dict(q=A + 4), INV), (dict(ldq=36), INV), (dict(n=0x7fffffff, ldx=1 << 40, ldq=1 << 40, lds=1 << 40), UNS),
    (dict(rows=0x7fffffff, n=65536, ldx=65536, ldq=1 << 20, lds=1 << 20), UNS), (dict(rows=0), OK)])
def test_quantize_mx(kw, rc):
    assert call(_lib.lib().dlk_quantize_mx, QUANT, **kw) == rc


DEQUANT = dict(q=A, ldq=32, scale=A, lds=2, table=2, ids=None, rows=2, n=64, format=FP4, out=A, dtype=_lib.BF16, ld=64,
               stream=None)


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), INV), (dict(scale=None), INV), (dict(out=None), INV), (dict(rows=-1), INV), (dict(table=-1), INV),
    (dict(n=0), INV), (dict(ld=63), INV), (dict(ldq=24), INV), (dict(format=FP6, ldq=40), INV), (dict(lds=1), INV),
    (dict(dtype=5), INV), (dict(format=7), INV), (dict(out=A + 1), INV), (dict(out=A + 2, dtype=_lib.F32), INV),
    (dict(q=A + 2), INV), (dict(ldq=34), INV), (dict(rows=3), INV), (dict(table=0, ids=A), INV), (dict(ids=A + 2), INV),
    (dict(n=0x7fffffff, ld=1 << 40, ldq=1 << 40, lds=1 << 40), UNS), (dict(rows=0), OK), (dict(rows=0, table=0), OK)])
def test_dequantize_mx(kw, rc):
    assert call(_lib.lib().dlk_dequantize_mx, DEQUANT, **kw) == rc


LOGITS = dict(x=A, format=FP4, ldx=32, x_scale=A, ldxs=16, w=A, ldw=32, w_scale=A, ldws=16, rows=2, vocab=100, n=64,
              softcap=0.0, logits=A, ld=100, stream=None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), INV), (dict(w=None), INV), (dict(x_scale=None), INV), (dict(w_scale=None), INV),
    (dict(logits=None), INV), (dict(rows=-1), INV), (dict(vocab=0), INV), (dict(n=0), INV), (dict(format=2), INV),
    (dict(ldx=16), INV), (dict(format=FP6), INV), (dict(ldw=16), INV), (dict(ldxs=2), INV), (dict(ldws=15), INV),
    (dict(ld=99), INV), (dict(x=A + 8), INV), (dict(x=A + 4, format=FP6, ldx=48), INV), (dict(ldx=40), INV),
    (dict(w=A + 8), INV), (dict(x_scale=A + 4), INV), (dict(w_scale=A + 1), INV), (dict(ldws=24), INV),
    (dict(logits=A + 2), INV), (dict(softcap=float("inf")), INV), (dict(softcap=float("nan")), INV),
    (dict(n=1 << 30, ldx=1 << 40, ldw=1 << 40, ldxs=1 << 40, ldws=1 << 40), UNS),
    (dict(vocab=0x7fffffff, ld=1 << 40), UNS), (dict(vocab=1 << 30, rows=1 << 10, ld=1 << 30), UNS), (dict(rows=0), OK)])
def test_logits_mx(kw, rc):
    assert call(_lib.lib().dlk_logits_mx, LOGITS, **kw) == rc


def score(rows=1, vocab=100, batch=(), **prm):
    b = _lib.LogprobBatch(logits=A, ld=vocab, tokens=A, out_logprobs=A, out_stats=A, out_top_ids=A, out_top_logprobs=A)
    for k, v in dict(batch).items():
        setattr(b, k, v)
    p = _lib.LogprobParams(**dict(dict(n_given=1, n_top=2, temperature=1.0), **prm))
    return _lib.lib().dlk_token_logprobs(C.byref(b), rows, vocab, C.byref(p), None)


def grad(rows=1, vocab=100, batch=(), **prm):
    b = _lib.LogprobGradBatch(logits=A, ld=vocab, tokens=A, stats=A, grad_logprobs=A, grad=A + 4096, ld_grad=vocab)
    for k, v in dict(batch).items():
        setattr(b, k, v)
    p = _lib.LogprobParams(**dict(dict(n_given=1, n_top=0, temperature=1.0), **prm))
    return _lib.lib().dlk_token_logprobs_grad(C.byref(b), rows, vocab, C.byref(p), None)


BOTH = [
    (dict(rows=-1), INV), (dict(vocab=0), INV), (dict(batch=dict(logits=None)), INV), (dict(batch=dict(ld=99)), INV),
    (dict(batch=dict(dtype=3)), INV), (dict(n_given=-1), INV), (dict(batch=dict(tokens=None)), INV),
    (dict(batch=dict(mask=A, mask_ld=3)), INV), (dict(temperature=0.0), INV), (dict(temperature=-1.0), INV),
    (dict(temperature=float("nan")), INV), (dict(temperature=float("inf")), INV), (dict(temperature=1e-31), INV),
    (dict(batch=dict(logits=A + 2)), INV), (dict(batch=dict(logits=A + 1, dtype=_lib.BF16)), INV),
    (dict(n_given=65), UNS), (dict(vocab=0x7fffffff), UNS), (dict(rows=0), OK),
    (dict(rows=0, n_given=0, batch=dict(tokens=None)), OK)]


@pytest.mark.parametrize("kw,rc", BOTH + [
    (dict(batch=dict(out_logprobs=None)), INV), (dict(batch=dict(out_top_ids=None)), INV),
    (dict(batch=dict(out_top_logprobs=None)), INV), (dict(n_top=-1), INV), (dict(n_top=65), UNS),
    (dict(batch=dict(out_stats=A + 2)), INV)])
def test_token_logprobs(kw, rc):
    assert score(**kw) == rc


@pytest.mark.parametrize("kw,rc", BOTH + [
    (dict(batch=dict(stats=None)), INV), (dict(batch=dict(grad=None)), INV), (dict(batch=dict(grad_logprobs=None)), INV),
    (dict(batch=dict(ld_grad=99)), INV), (dict(batch=dict(grad=A + 2)), INV),
    (dict(rows=2, batch=dict(grad=A, ld_grad=104)), INV)])
def test_token_logprobs_grad(kw, rc):
    assert grad(**kw) == rc


def test_null_structures():
    L = _lib.lib()
    p = _lib.LogprobParams(1, 0, 1.0)
    assert L.dlk_token_logprobs(None, 1, 1, C.byref(p), None) == INV
    assert L.dlk_token_logprobs(C.byref(_lib.LogprobBatch()), 1, 1, None, None) == INV
    assert L.dlk_token_logprobs_grad(None, 1, 1, C.byref(p), None) == INV
    assert L.dlk_token_logprobs_grad(C.byref(_lib.LogprobGradBatch()), 1, 1, None, None) == INV


# ---- the Python functions ----------------------------------------------------------

def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def f32(*shape):
    return torch.zeros(shape)


@pytest.mark.parametrize("fn", [
    lambda: api.quantize_mx(f32(4, 64)),                                           # not on a GPU
    lambda: api.quantize_mx(f32(4, 64).double()),
    lambda: api.quantize_mx(f32(64)),
    lambda: api.quantize_mx(f32(4, 64), "fp8"),
    lambda: api.quantize_mx(f32(64, 4).t()),
    lambda: api.quantize_mx(f32(4, 64), q=u8(4, 48)),
    lambda: api.quantize_mx(f32(4, 64), "fp6", q=u8(4, 32)),
    lambda: api.quantize_mx(f32(4, 64), scale=u8(4, 3)),
    lambda: api.quantize_mx(f32(4, 64), scale=u8(3, 2)),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2)),                                # not on a GPU
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 3)),
    lambda: api.dequantize_mx(u8(4, 32), u8(3, 2)),
    lambda: api.dequantize_mx(u8(4, 64), u8(4, 2)),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), n=32),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), n=65),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), ids=torch.zeros(3, dtype=torch.int64)),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), dtype=torch.float64),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), out=f32(4, 63)),
    lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), ids=i32(3), out=f32(4, 64)),
    lambda: api.logits_mx(u8(2, 32), u8(2, 2), u8(9, 32), u8(9, 2)),               # not on a GPU
    lambda: api.logits_mx(u8(2, 32), u8(2, 2), u8(9, 48), u8(9, 2)),               # weights of 6 bits
    lambda: api.logits_mx(u8(2, 32), u8(2, 2), u8(9, 48), u8(9, 3)),
    lambda: api.logits_mx(u8(2, 32), u8(2, 2), u8(9, 32), u8(9, 2), out=f32(2, 8)),
    lambda: api.logits_mx(u8(2, 32).char(), u8(2, 2), u8(9, 32), u8(9, 2)),
    lambda: api.logits_mx(u8(2, 48)[:, :32], u8(2, 16)[:, :2], u8(9, 32), u8(9, 2)),              # packed scales
    lambda: api.logits_mx(u8(2, 40)[:, :32], u8(2, 16)[:, :2], u8(9, 32), u8(9, 16)[:, :2]),
    lambda: api.logits_mx(u8(2, 32), u8(2, 16)[:, :2], u8(9 * 32 + 8)[8:].view(9, 32), u8(9, 16)[:, :2]),
    lambda: api.quantize_mx(f32(4, 64), q=u8(4, 36)[:, :32]),
    lambda: api.dequantize_mx(u8(4, 36)[:, :32], u8(4, 2)),
    lambda: api.token_logprobs(f32(2, 9)),                                         # not on a GPU
    lambda: api.token_logprobs(f32(2, 9).double()),
    lambda: api.token_logprobs(f32(2, 9), torch.zeros(2, dtype=torch.int64)),
    lambda: api.token_logprobs(f32(2, 9), i32(3)),
    lambda: api.token_logprobs(f32(2, 9), i32(2, 1, 1)),
    lambda: api.token_logprobs(f32(2, 9), i32(4, 2)[:, 0][::2]),
    lambda: api.token_logprobs(f32(2, 9), top=-1),
    lambda: api.token_logprobs(f32(2, 9), top=1 << 32),
    lambda: api.token_logprobs(f32(2, 33), mask=i32(2, 1)),
    lambda: api.token_logprobs(f32(2, 9), mask=i32(1, 1)),
    lambda: api.token_logprobs(f32(2, 9), mask=i32(1, 1), mask_row=i32(1)),
    lambda: api.token_logprobs(f32(2, 9), i32(2), out=dict(stats=f32(2, 4), logprobs=f32(1))),
    lambda: api.token_logprobs(f32(2, 9), status=f32(1)),
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), f32(2)),         # not on a GPU
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 3), f32(2)),
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), None),
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), f32(1)),
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), f32(2), grad_entropy=f32(1)),
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), f32(2), out=f32(2, 8)),
    lambda: api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), f32(2), out=f32(2, 9).half()),
])
def test_python(fn):
    with pytest.raises(ValueError):
        fn()


@pytest.fixture
def on_no_device(monkeypatch):
    """CPU or meta tensors taken for the GPU's, calls recorded and not made; returns what was called."""
    calls = []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(api, "_call", lambda dev, stream, what, fn, *args: calls.append((what, stream, args)))
    return calls


def test_counts_past_32_bits(on_no_device):
    """What ctypes would cut to its low 32 bits is refused."""
    big = 1 << 32
    meta = lambda *shape, **kw: torch.empty(shape, device="meta", **kw)
    for bad in (lambda: api.quantize_mx(meta(big + 1, 32)), lambda: api.quantize_mx(meta(1, big + 32)),
                lambda: api.dequantize_mx(u8(4, 32), u8(4, 2), ids=meta(big + 1, dtype=torch.int32)),
                lambda: api.logits_mx(meta(big + 1, 16, dtype=torch.uint8), meta(big + 1, 1, dtype=torch.uint8),
                                      u8(9, 16), u8(9, 1)),
                lambda: api.token_logprobs(meta(big + 1, 9)), lambda: api.token_logprobs(meta(1, big + 9)),
                lambda: api.token_logprobs(f32(2, 9), top=big + 1)):
        with pytest.raises(ValueError):
            bad()
    assert on_no_device == []


def test_table_without_rows(on_no_device):
    """Has no row to give zeros for: refused with ids as in C, nothing to do without any."""
    with pytest.raises(ValueError):
        api.dequantize_mx(u8(0, 32), u8(0, 2), ids=i32(3))
    assert api.dequantize_mx(u8(0, 32), u8(0, 2), ids=i32(0)).shape == api.dequantize_mx(u8(0, 32), u8(0, 2)).shape == (0, 64)
    assert on_no_device == []


@pytest.mark.parametrize("current,stream,made_on", [(111, 222, 222), (111, 0, 0), (111, 111, None), (111, None, None)])
def test_outputs_are_made_on_the_calls_stream(on_no_device, monkeypatch, current, stream, made_on):
    """Outputs that a call makes come from the memory of the stream that writes them."""
    import contextlib
    now, made = [None], []

    @contextlib.contextmanager
    def on(s):
        before, now[0] = now[0], s
        yield
        now[0] = before
    empty = torch.empty
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda at, device=None: at)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: current, raising=False)
    # (16-byte aligned, as the allocator's)
    aligned = torch.zeros(1 << 16, dtype=torch.uint8)
    aligned = aligned[-aligned.data_ptr() % 64:]
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: made.append(now[0]) or empty(*a, **kw))
    q, s = aligned[:64].view(2, 32), aligned[64:96].view(2, 16)[:, :2]
    api.quantize_mx(f32(4, 64), q=aligned[:128].view(4, 32), stream=stream)                         # the scales
    api.dequantize_mx(q, s, stream=stream)
    api.logits_mx(q, s, q, s, stream=stream)
    api.token_logprobs(f32(2, 9), i32(2), top=3, stream=stream)                                   # four
    api.token_logprobs_grad(f32(2, 9), i32(2), f32(2, 4), f32(2), stream=stream)
    assert [s for _, s, _ in on_no_device] == [stream] * 5
    assert made == [made_on] * 8 and now == [None]
