"""What dlk_quantize_rows, dlk_logits_i8, dlk_beam_select and dlk_beam_reorder refuse, before any device work: through
the C entry points with addresses that are never read, and through the Python functions with CPU tensors."""
import ctypes as C

import pytest
import torch

from diskllm_amd import _lib, api

A = 1 << 20                       # some 16-byte aligned address
INV, UNS, OK = _lib.DLK_ERR_INVALID, _lib.DLK_ERR_UNSUPPORTED, _lib.DLK_OK


def call(fn, base, **kw):
    """fn with base's arguments (in order), some of them changed."""
    a = dict(base)
    assert set(kw) <= set(a)
    a.update(kw)
    return fn(*a.values())


QUANT = dict(x=A, dtype=_lib.BF16, ldx=64, rows=2, n=64, q=A, ldq=64, scale=A, stream=None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), INV), (dict(q=None), INV), (dict(scale=None), INV), (dict(rows=-1), INV), (dict(n=0), INV),
    (dict(ldx=63), INV), (dict(ldq=63), INV), (dict(dtype=3), INV), (dict(dtype=-1), INV), (dict(x=A + 1), INV),
    (dict(x=A + 2, dtype=_lib.F32), INV), (dict(scale=A + 2), INV),
    (dict(n=0x7fffffff, ldx=1 << 40, ldq=1 << 40), UNS), (dict(rows=0), OK),
    (dict(n=2000, ldx=2000, ldq=2000, rows=1 << 24), UNS), (dict(rows=1 << 26), UNS)])      # 2^32 threads
def test_quantize_rows(kw, rc):
    assert call(_lib.lib().dlk_quantize_rows, QUANT, **kw) == rc


@pytest.mark.parametrize("n,most", [(64, 4 * 0xffffff), (1024, 4 * 0xffffff), (1025, 0xffffff)])
@pytest.mark.parametrize("over", [1, 2, 3, 4])
def test_quantize_rows_past_a_launch(n, most, over):
    """Four rows to a workgroup of 256 threads up to 1,024 entries, one past that: 2^24 workgroups are no launch."""
    assert call(_lib.lib().dlk_quantize_rows, QUANT, rows=most + over, n=n, ldx=n, ldq=n) == UNS


LOGITS = dict(x=A, ldx=64, x_scale=A, w=A, ldw=64, w_scale=A, rows=2, vocab=100, n=64, softcap=0.0, logits=A, ld=100,
              stream=None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), INV), (dict(w=None), INV), (dict(x_scale=None), INV), (dict(w_scale=None), INV),
    (dict(logits=None), INV), (dict(rows=-1), INV), (dict(vocab=0), INV), (dict(n=0), INV), (dict(ldx=63), INV),
    (dict(ldw=63), INV), (dict(ld=99), INV), (dict(logits=A + 2), INV), (dict(w_scale=A + 1), INV),
    (dict(n=131072, ldx=131072, ldw=131072), UNS), (dict(softcap=float("inf")), INV), (dict(vocab=0x7fffffff, ld=1 << 40), UNS), (dict(rows=0), OK),
    (dict(vocab=1 << 30, ld=1 << 30), UNS),
    (dict(softcap=float("nan")), INV), (dict(softcap=float("-inf")), INV)])
def test_logits_i8(kw, rc):
    assert call(_lib.lib().dlk_logits_i8, LOGITS, **kw) == rc


def select(groups=1, vocab=100, batch=(), **prm):
    b = _lib.BeamBatch(logits=A, ld=vocab, scores=A + 4096, out_tokens=A, out_parents=A, out_scores=A)
    for k, v in dict(batch).items():
        setattr(b, k, v)
    p = _lib.BeamParams(beams=4, n_out=4, eos_id=-1, length_penalty=0.0, repeat_penalty=1.0)
    for k, v in prm.items():
        setattr(p, k, v)
    return _lib.lib().dlk_beam_select(C.byref(b), groups, vocab, C.byref(p), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(groups=-1), INV), (dict(vocab=0), INV), (dict(batch=dict(logits=None)), INV),
    (dict(batch=dict(logits=A + 2)), INV), (dict(batch=dict(ld=99)), INV), (dict(batch=dict(out_tokens=None)), INV),
    (dict(batch=dict(out_parents=None)), INV), (dict(batch=dict(out_scores=None)), INV), (dict(beams=0), INV),
    (dict(n_out=0), INV), (dict(batch=dict(hist_off=A)), INV), (dict(batch=dict(hist_ids=A)), INV),
    (dict(batch=dict(mask=A, mask_ld=3)), INV), (dict(eos_id=100), INV), (dict(eos_id=-2), INV),
    (dict(batch=dict(finished=A)), INV), (dict(length_penalty=float("nan")), INV),
    (dict(length_penalty=float("inf")), INV), (dict(length_penalty=17.0), INV), (dict(max_history=-1), INV),
    (dict(beams=65), UNS), (dict(n_out=65), UNS), (dict(max_history=65536), UNS),
    (dict(vocab=0x7fffffff), UNS), (dict(groups=0x7fffffff), UNS), (dict(groups=0), OK),
    # an output that is its own input
    (dict(batch=dict(out_scores=A, scores=A)), INV), (dict(batch=dict(out_lengths=A, lengths=A)), INV),
    (dict(batch=dict(out_finished=A, finished=A), eos_id=3), INV)])
def test_beam_select(kw, rc):
    assert select(**kw) == rc
    assert _lib.lib().dlk_beam_select(None, 1, 100, None, None) == INV


def state(**kw):
    s = _lib.BeamState(src=A, dst=A, bytes=64, src_row=128, src_outer=4096, src_inner=64, dst_row=128, dst_outer=4096,
                       dst_inner=64, n_outer=2, n_inner=2)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def reorder(parents=A, groups=2, beams=4, n_out=4, states=(), history=None):
    arr = (_lib.BeamState * max(1, len(states)))(*states)
    return _lib.lib().dlk_beam_reorder(parents, groups, beams, n_out, arr, len(states), history, None)


FAR = A + (1 << 20)


@pytest.mark.parametrize("kw,rc", [
    (dict(parents=None), INV), (dict(groups=-1), INV), (dict(beams=0), INV), (dict(n_out=0), INV),
    (dict(beams=65), UNS), (dict(n_out=65), UNS), (dict(groups=0x7fffffff), UNS), (dict(groups=0), OK),
    (dict(states=[state(src=None)]), INV), (dict(states=[state(dst=None)]), INV), (dict(states=[state(bytes=-1)]), INV),
    (dict(states=[state(src_row=-128)]), INV), (dict(states=[state(dst_inner=-64)]), INV),
    (dict(states=[state(n_outer=-1)]), INV),
    # in place: one layout, as many rows after as before
    (dict(states=[state()], n_out=3), INV), (dict(states=[state(src_row=256)]), INV),
    # destinations that overlap themselves
    (dict(states=[state(bytes=65)]), INV), (dict(states=[state(src_row=64, dst_row=64)]), INV),
    (dict(states=[state(src_outer=512, dst_outer=512)]), INV),
    # more than a launch takes
    (dict(states=[state(n_outer=1 << 23, n_inner=1, src_outer=1024, dst_outer=1024)]), UNS),
    # one buffer twice, in place or behind another source; two that change places
    (dict(states=[state(), state()]), INV), (dict(states=[state(dst=FAR), state(src=A - 8192, dst=FAR)]), INV),
    (dict(states=[state(dst=FAR), state(src=FAR, dst=A)]), INV), (dict(states=[state(), state(dst=FAR)]), INV),
    # two buffers that overlap
    (dict(states=[state(dst=A + 4096)]), INV), (dict(states=[state(dst=A - 4096)]), INV)])
def test_beam_reorder(kw, rc):
    assert reorder(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(off=None), INV), (dict(ids=None), INV), (dict(out_off=None), INV), (dict(out_ids=None), INV),
    (dict(max_history=0), INV), (dict(out_off=A), INV), (dict(out_ids=A + 256), INV),
    (dict(max_history=0x10000000), UNS), (dict(groups=1 << 22, max_history=1), UNS)])
def test_beam_history(kw, rc):
    h = _lib.BeamHistory(A, A + 256, A + 512, 16, FAR, FAR + 256)
    groups = kw.get("groups", 2)
    for k, v in kw.items():
        if k != "groups":
            setattr(h, k, v)
    assert reorder(groups=groups, history=C.byref(h)) == rc


def test_python_refusals():
    f, i, b = torch.float32, torch.int32, torch.int8
    z = torch.zeros
    for bad in (lambda: api.quantize_rows(z(4, 8, dtype=torch.float64)), lambda: api.quantize_rows(z(8)),
                lambda: api.quantize_rows(z(8, 4).t()), lambda: api.quantize_rows(z(4, 8), z(4, 7, dtype=b)),
                lambda: api.quantize_rows(z(4, 8), scale=z(3)), lambda: api.quantize_rows(z(4, 8)),
                lambda: api.logits_i8(z(4, 8, dtype=b), z(4), z(9, 7, dtype=b), z(9)),
                lambda: api.logits_i8(z(4, 8, dtype=b), z(4), z(9, 8), z(9)),
                lambda: api.logits_i8(z(4, 8, dtype=b), z(3), z(9, 8, dtype=b), z(9)),
                lambda: api.logits_i8(z(4, 8, dtype=b), z(4), z(9, 8, dtype=b), z(9), out=z(4, 8)),
                lambda: api.logits_i8(z(4, 8, dtype=b), z(4), z(9, 8, dtype=b), z(9)),
                lambda: api.beam_select(z(7, 30), 4, 4), lambda: api.beam_select(z(8, 30, dtype=torch.float16), 4, 4),
                lambda: api.beam_select(z(8, 30), 4, 4, scores=z(7)),
                lambda: api.beam_select(z(8, 30), 4, 4, finished=z(8)),
                lambda: api.beam_select(z(8, 70), 4, 4, mask=z(8, 2, dtype=i)),
                lambda: api.beam_select(z(8, 70), 4, 4, mask=z(7, 3, dtype=i)),
                lambda: api.beam_select(z(8, 30), 4, 4, hist_off=z(8, dtype=i), hist_ids=z(8, dtype=i)),
                lambda: api.beam_select(z(8, 30), 4, 4),
                lambda: api.beam_state(z(2, 4, 8).transpose(1, 2)), lambda: api.beam_state(z(4, 8), z(4, 9)),
                lambda: api.beam_state(z(4, 8), z(4, 8, dtype=i)), lambda: api.beam_state(z(4, 8, 2), length_dim=0),
                lambda: api.beam_state(z(4, 8, 2), length_dim=1, length=9),
                lambda: api.beam_reorder(z(7, dtype=i), 4, 4),
                lambda: api.beam_reorder(z(8, dtype=i), 4, 4, [api.beam_state(z(7, 3))]),
                lambda: api.beam_reorder(z(8, dtype=i), 4, 4, history=api.beam_history(
                    z(9, dtype=i), z(8, dtype=i), z(8, dtype=i), 4, z(9, dtype=i), z(31, dtype=i))),
                lambda: api.beam_reorder(z(8, dtype=i), 4, 4, [api.beam_state(z(8, 3))])):
        with pytest.raises(ValueError):
            bad()


def test_state_layouts():
    """A cache's strides as beam_state takes them."""
    c = torch.zeros((3, 8, 2, 16, 4), dtype=torch.bfloat16)
    s = api.beam_state(c, row_dim=1, length_dim=3, length=5)
    assert (s.bytes, s.n_outer, s.n_inner) == (5 * 4 * 2, 3, 2)
    assert (s.src_outer, s.src_row, s.src_inner) == (8 * 2 * 16 * 4 * 2, 2 * 16 * 4 * 2, 16 * 4 * 2)
    assert s.src == s.dst == c.data_ptr() and s.dst_row == s.src_row
    r = api.beam_state(torch.zeros((8, 40), dtype=torch.uint8))
    assert (r.bytes, r.n_outer, r.n_inner, r.src_row) == (40, 1, 1, 40)
    one = api.beam_state(torch.zeros(8))
    assert (one.bytes, one.src_row) == (4, 4)
    # [rows, layers, heads, room, width]: layers and heads in one stride
    d = api.beam_state(torch.zeros((8, 3, 2, 16, 4)), length_dim=3, length=16)
    assert (d.bytes, d.n_outer, d.n_inner, d.src_inner) == (16 * 4 * 4, 1, 6, 16 * 4 * 4)
    assert api.beam_state(c, row_dim=1, length_dim=3, length=0).bytes == 0
    # a single row or head whose stride says nothing
    one = torch.zeros((3, 8, 2, 16, 4)).as_strided((3, 1, 1, 16, 4), (64, 7, 5, 4, 1))
    assert one.is_contiguous()
    u = api.beam_state(one, row_dim=1, length_dim=3, length=5)
    assert (u.bytes, u.n_outer, u.n_inner, u.src_outer) == (5 * 4 * 4, 3, 1, 64 * 4)
    # rows that lie apart
    v = api.beam_state(torch.zeros((8, 3, 40))[:, 1])
    assert (v.bytes, v.n_outer, v.n_inner, v.src_row) == (160, 1, 1, 480)


@pytest.fixture
def on_no_device(monkeypatch):
    """CPU or meta tensors taken for the GPU's, calls recorded and not made; returns what was called."""
    calls = []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(api, "_call", lambda dev, stream, what, fn, *args: calls.append((what, stream, args)))
    return calls


def test_counts_past_32_bits(on_no_device):
    """What ctypes would cut to its low 32 bits is refused."""
    i, big = torch.int32, 1 << 32
    z = torch.zeros
    meta = lambda *shape, **kw: torch.empty(shape, device="meta", **kw)
    spread = lambda n, m: torch.empty_strided((n, 4, m), (8 * m, 2 * m, 1), device="meta", dtype=torch.uint8)
    hist = lambda n: api.beam_history(z(9, dtype=i), z(8, dtype=i), None, n, z(9, dtype=i), z(99, dtype=i))
    for bad in (lambda: api.beam_state(meta(big + 1, 4, dtype=torch.uint8), row_dim=1),
                lambda: api.beam_state(meta(4, big + 1, 1, dtype=torch.uint8), length_dim=2),
                lambda: api.beam_state(spread(big + 1, 2), row_dim=1),
                lambda: hist(big + 1), lambda: hist(-big + 8),
                lambda: api.beam_select(z(8, 30), 4, 4, max_history=big + 8),
                lambda: api.beam_select(z(8, 30), 4, 4, eos_id=big + 8),
                lambda: api.beam_select(z(8, 30), 4, 4, eos_id=-big + 8),
                lambda: api.beam_select(z(8, 30), 4, 4, order=big + 1),
                lambda: api.beam_select(z(8, 30), 4, 4, order=-1),
                lambda: api.beam_select(z(0, 30), big + 4, 4), lambda: api.beam_select(z(0, 30), 4, big + 4),
                lambda: api.beam_reorder(meta(big + 4, dtype=i), 1, 1), lambda: api.beam_reorder(z(0, dtype=i), 4, big + 4)):
        with pytest.raises(ValueError):
            bad()
    assert on_no_device == []
    # what fits still goes through
    assert api.beam_state(meta((1 << 31) - 1, 4, dtype=torch.uint8), row_dim=1).n_outer == (1 << 31) - 1
    api.beam_select(z(8, 30), 4, 4, max_history=65535, eos_id=29, order=0xffffffff)
    assert len(on_no_device) == 1


@pytest.mark.parametrize("current,stream,made_on", [(111, 222, 222), (111, 0, 0), (0, 222, 222), (111, 111, None),
                                                    (111, None, None), (0, 0, None)])
def test_outputs_are_made_on_the_calls_stream(on_no_device, monkeypatch, current, stream, made_on):
    """Outputs that a call makes come from the memory of the stream that writes them: a block of the current stream's
    may still be in use there, and goes back to it while the kernel writes."""
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
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: made.append(now[0]) or empty(*a, **kw))
    b = torch.int8
    api.quantize_rows(torch.zeros(4, 8), stream=stream)
    api.quantize_rows(torch.zeros(4, 8), q=torch.zeros((4, 8), dtype=b), stream=stream)
    api.logits_i8(torch.zeros((4, 8), dtype=b), torch.zeros(4), torch.zeros((9, 8), dtype=b), torch.zeros(9), stream=stream)
    api.beam_select(torch.zeros(8, 30), 4, 4, stream=stream)
    assert [s for _, s, _ in on_no_device] == [stream] * 4
    assert made == [made_on] * 7 and now == [None]
