"""Python host side of the batched sampling path.

Mirrors the C ABI of include/diskllm_amd.h one-to-one; torch tensors are only
device-memory and stream plumbing.  Every call goes through libdiskllm_amd.so.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import _lib
from .workloads import Workload


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dev(a: np.ndarray, device) -> torch.Tensor:
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    elif a.dtype == np.uint64:
        a = a.view(np.int64)
    return torch.from_numpy(a).to(device)


def stream_handle(device=None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


@dataclass
class DeviceBatch:
    """A workload's inputs resident in HBM plus output buffers."""
    w: Workload
    logits: torch.Tensor
    seeds: torch.Tensor            # int64 view of the per-row uint64 seeds (never mutated)
    rng: torch.Tensor              # int64 view of the per-row xorshift states (mutated)
    hist_off: Optional[torch.Tensor]
    hist_ids: Optional[torch.Tensor]
    mask: Optional[torch.Tensor]
    mask_row: Optional[torch.Tensor]
    out_ids: torch.Tensor
    cand_ids: Optional[torch.Tensor]
    cand_probs: Optional[torch.Tensor]
    cand_logprobs: Optional[torch.Tensor]
    status: torch.Tensor

    def reset_rng(self) -> None:
        self.rng.copy_(self.seeds)


def dfa_masks(offsets, data, trans, states, vocab: int, eos_id: int = -1, accept: int = 0,
              device="cuda", stream: Optional[int] = None) -> torch.Tensor:
    """Packed allow-masks [len(states), ceil(V/32)] (int32 view of uint32 words)."""
    W = (vocab + 31) // 32
    t_off = offsets if isinstance(offsets, torch.Tensor) else _dev(np.asarray(offsets, np.uint32), device)
    t_dat = data if isinstance(data, torch.Tensor) else _dev(np.asarray(data, np.uint8), device)
    tr = np.ascontiguousarray(trans, np.uint8)
    t_tr = _dev(tr, device)
    t_st = states if isinstance(states, torch.Tensor) else _dev(np.asarray(states, np.int32), device)
    out = torch.empty((t_st.numel(), W), dtype=torch.int32, device=device)
    rc = _lib.lib().dlk_dfa_mask(t_off.data_ptr(), t_dat.data_ptr(), vocab, t_tr.data_ptr(), tr.shape[0],
                                 t_st.data_ptr(), t_st.numel(), eos_id, accept & 0xFFFFFFFFFFFFFFFF, out.data_ptr(),
                                 W, stream if stream is not None else stream_handle())
    _lib.check(rc, "dlk_dfa_mask")
    return out


def to_device(w: Workload, device="cuda", rows: Optional[list] = None) -> DeviceBatch:
    sel = list(range(w.rows)) if rows is None else list(rows)
    lg = _dev(np.ascontiguousarray(w.logits[sel]), device)
    seeds = _dev(np.ascontiguousarray(w.seeds[sel]), device)
    hoff = hids = None
    if w.hist_ids is not None:
        lists = [w.hist_ids[w.hist_off[r]:w.hist_off[r + 1]] for r in sel]
        off = np.zeros(len(sel) + 1, np.int32)
        off[1:] = np.cumsum([len(x) for x in lists])
        ids = np.concatenate(lists).astype(np.int32) if lists else np.zeros(0, np.int32)
        hoff, hids = _dev(off, device), _dev(ids if ids.size else np.zeros(1, np.int32), device)
    mask = mask_row = None
    if w.mask is not None:
        mask = _dev(np.ascontiguousarray(w.mask[sel]), device)
    elif w.dfa is not None and w.dfa_states is not None:
        n_states = w.dfa.trans.shape[0]
        mask = dfa_masks(w.dfa.offsets, w.dfa.data, w.dfa.trans, np.arange(n_states, dtype=np.int32), w.vocab,
                         w.dfa.eos_id, w.dfa.accept, device)
        mask_row = _dev(np.asarray(w.dfa_states[sel], np.int32), device)
    n = len(sel)
    no = w.n_out
    return DeviceBatch(
        w=w, logits=lg, seeds=seeds, rng=seeds.clone(), hist_off=hoff, hist_ids=hids, mask=mask, mask_row=mask_row,
        out_ids=torch.full((n,), -7, dtype=torch.int32, device=device),
        cand_ids=torch.zeros((n, no), dtype=torch.int32, device=device) if no else None,
        cand_probs=torch.zeros((n, no), dtype=torch.float32, device=device) if no else None,
        cand_logprobs=torch.zeros((n, no), dtype=torch.float32, device=device) if no else None,
        status=torch.zeros(1, dtype=torch.int32, device=device))


def params_of(w: Workload, max_history: int = 0, path: int = 0) -> _lib.SampleParams:
    mh = max_history
    if mh <= 0 and w.hist_off is not None and len(w.hist_off) > 1:
        mh = int(np.max(np.diff(w.hist_off)))
    return _lib.SampleParams(w.temperature, w.top_k, w.top_p, w.min_p, w.repeat_penalty, w.frequency_penalty,
                             w.presence_penalty, w.order, max(mh, 1), w.n_out, path, w.softcap)


def batch_struct(db: DeviceBatch) -> _lib.Batch:
    w = db.w
    return _lib.Batch(
        logits=db.logits.data_ptr(), ld=db.logits.shape[1], hist_off=_ptr(db.hist_off), hist_ids=_ptr(db.hist_ids),
        mask=_ptr(db.mask), mask_ld=(db.mask.shape[1] if db.mask is not None else 0), mask_row=_ptr(db.mask_row),
        rng=db.rng.data_ptr(), out_ids=db.out_ids.data_ptr(), out_cand_ids=_ptr(db.cand_ids),
        out_cand_probs=_ptr(db.cand_probs), out_cand_logprobs=_ptr(db.cand_logprobs), status=db.status.data_ptr())


def sample(db: DeviceBatch, params: Optional[_lib.SampleParams] = None, stream: Optional[int] = None) -> None:
    """One dlk_sample call over the batch (asynchronous on the stream)."""
    w = db.w
    p = params if params is not None else params_of(w)
    b = batch_struct(db)
    rc = _lib.lib().dlk_sample(C.byref(b), db.logits.shape[0], w.vocab, C.byref(p),
                               stream if stream is not None else stream_handle())
    _lib.check(rc, "dlk_sample")


def sampler(db: DeviceBatch, params: Optional[_lib.SampleParams] = None, stream: Optional[int] = None):
    """A callable that makes the dlk_sample call of sample() with its argument
    structures built once: a loop of calls then costs the C call alone (timing
    loops; the batch's buffers must stay where they are)."""
    w = db.w
    p = params if params is not None else params_of(w)
    b = batch_struct(db)
    f = _lib.lib().dlk_sample
    rows, vocab = db.logits.shape[0], w.vocab
    sh = stream if stream is not None else stream_handle()
    bp, pp = C.byref(b), C.byref(p)

    def run() -> None:
        rc = f(bp, rows, vocab, pp, sh)
        if rc != 0:
            _lib.check(rc, "dlk_sample")
    run.keep = (b, p)
    return run


def results(db: DeviceBatch) -> dict:
    torch.cuda.synchronize()
    out = dict(ids=db.out_ids.cpu().numpy(), states=db.rng.cpu().numpy().view(np.uint64),
               status=int(db.status.cpu().item()))
    if db.cand_ids is not None:
        out.update(cand_ids=db.cand_ids.cpu().numpy(), cand_probs=db.cand_probs.cpu().numpy(),
                   cand_logprobs=db.cand_logprobs.cpu().numpy())
    return out


# ---- 8-bit logits and beam search ------------------------------------------------
# Tensors on one device, the call on that device's current stream unless `stream` (a raw
# handle) says otherwise; what does not fit raises ValueError before anything is launched.
# Tensors that a call makes belong to the stream it runs on, as those made under
# torch.cuda.stream: another stream waits for it first, and record_stream tells the
# allocator where they outlive that wait.

_F32, _I32, _I8, _U8 = torch.float32, torch.int32, torch.int8, torch.uint8
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


_WIDE = "{}: integers of 32 bits are wanted"          # (of a C int ctypes keeps the low bits)


def _rows2d(t: torch.Tensor, dev: int, dtype, what: str):
    """(rows, n, row stride) of a [rows, n] tensor whose rows are contiguous (dtype None: any)."""
    if t.dim() != 2 or (dtype is not None and t.dtype is not dtype) or t.get_device() != dev:
        raise ValueError(f"{what}: [rows, n] of {dtype} on the call's device is wanted")
    rows, n = t.shape
    if rows > 0x7fffffff or n > 0x7fffffff:
        raise ValueError(f"{what}: more rows or entries than 32 bits count")
    ld, one = t.stride()
    if rows <= 1 and ld < n:
        ld = n
    if (one != 1 and n > 1) or ld < n:
        raise ValueError(f"{what}: contiguous rows that do not overlap are wanted")
    return rows, n, ld


def _flat(t: torch.Tensor, n: int, dev: int, dtype, what: str) -> int:
    """The address of at least n contiguous values."""
    if t.dtype is not dtype or t.numel() < n or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{what}: at least {n} contiguous values of {dtype} on the call's device are wanted")
    return t.data_ptr()


def _empty(shape, dtype, like: torch.Tensor, dev: int, stream) -> torch.Tensor:
    """An output on like's device, of the memory that belongs to the call's stream: the allocator gives a block to
    one stream at a time, so one of the current stream's might still be in use there, or given away again while
    the kernel on `stream` writes it."""
    if stream is None or dev < 0 or stream == torch._C._cuda_getCurrentRawStream(dev):
        return torch.empty(shape, dtype=dtype, device=like.device)
    on = torch.cuda.ExternalStream(stream, device=like.device) if stream else torch.cuda.default_stream(like.device)
    with torch.cuda.stream(on):
        return torch.empty(shape, dtype=dtype, device=like.device)


def _call(dev: int, stream, what: str, fn, *args) -> None:
    """fn(*args, stream) with device `dev` current (the kernels run there)."""
    if dev < 0:
        raise ValueError(f"{what}: tensors on the GPU are wanted")
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc != 0:
        _lib.check(rc, what)


def quantize_rows(x: torch.Tensor, q: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                  stream: Optional[int] = None):
    """(q int8 [rows, n], scale float32 [rows]) of x [rows, n] in float32, bfloat16 or float16: hidden states with a
    scale per token, or weights [vocab, n] with one per channel (dlk_quantize_rows)."""
    dt = _DTYPES.get(x.dtype)
    _want(dt is not None, "x: float32, bfloat16 or float16 is wanted")
    dev = x.get_device()
    rows, n, ldx = _rows2d(x, dev, None, "x")
    if q is None:
        ldq = (n + 15) // 16 * 16
        q = _empty((rows, ldq), _I8, x, dev, stream)
        if ldq != n:
            q = q[:, :n]
    else:
        q_rows, q_n, ldq = _rows2d(q, dev, _I8, "q")
        _want(q_rows == rows and q_n == n, "q: x's shape is wanted")
    if scale is None:
        scale = _empty(rows, _F32, x, dev, stream)
        at = scale.data_ptr()
    else:
        at = _flat(scale, rows, dev, _F32, "scale")
    if rows:
        _call(dev, stream, "dlk_quantize_rows", _lib.lib().dlk_quantize_rows, x.data_ptr(), dt, ldx, rows, n,
              q.data_ptr(), ldq, at)
    return q, scale


def logits_i8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, softcap: float = 0.0,
              out: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """Logits float32 [rows, vocab] of x int8 [rows, n] (x_scale [rows]) over w int8 [vocab, n] (w_scale [vocab]),
    soft-capped where softcap > 0 (dlk_logits_i8)."""
    dev = x.get_device()
    rows, n, ldx = _rows2d(x, dev, _I8, "x")
    V, w_n, ldw = _rows2d(w, dev, _I8, "w")
    _want(w_n == n, "x and w: rows of one length are wanted")
    if out is None:
        ld = (V + 63) // 64 * 64
        out = _empty((rows, ld), _F32, x, dev, stream)
        if ld != V:
            out = out[:, :V]
    else:
        o_rows, o_n, ld = _rows2d(out, dev, _F32, "out")
        _want(o_rows == rows and o_n == V, "out: [rows, vocab] is wanted")
    xs, ws = _flat(x_scale, rows, dev, _F32, "x_scale"), _flat(w_scale, V, dev, _F32, "w_scale")
    if rows:
        _call(dev, stream, "dlk_logits_i8", _lib.lib().dlk_logits_i8, x.data_ptr(), ldx, xs, w.data_ptr(), ldw, ws,
              rows, V, n, softcap, out.data_ptr(), ld)
    return out


def beam_select(logits: torch.Tensor, beams: int, n_out: int, *, scores: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, finished: Optional[torch.Tensor] = None,
                hist_off: Optional[torch.Tensor] = None, hist_ids: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, mask_row: Optional[torch.Tensor] = None, eos_id: int = -1,
                length_penalty: float = 0.0, repeat_penalty: float = 1.0, frequency_penalty: float = 0.0,
                presence_penalty: float = 0.0, order: int = _lib.ORDER_REP_FREQ_PRES, max_history: int = 0,
                out: Optional[dict] = None, status: Optional[torch.Tensor] = None,
                stream: Optional[int] = None) -> dict:
    """One step of a beam search over logits float32 [groups * beams, vocab] (dlk_beam_select): tokens, parents,
    lengths (int32), scores (float32) and finished (uint8) of the n_out best continuations of each group."""
    dev = logits.get_device()
    rows, V, ld = _rows2d(logits, dev, _F32, "logits")
    _want(beams > 0 and n_out > 0 and rows % beams == 0, "logits: whole groups of beams are wanted")
    if ((beams | n_out) >> 31 or order >> 32 or not -0x80000000 <= eos_id <= 0x7fffffff or
            not -0x80000000 <= max_history <= 0x7fffffff):
        raise ValueError(_WIDE.format("beam_select"))
    groups = rows // beams
    n = groups * n_out
    if out is None:
        i32 = _empty((3, n), _I32, logits, dev, stream)
        out = dict(tokens=i32[0], parents=i32[1], lengths=i32[2], scores=_empty(n, _F32, logits, dev, stream),
                   finished=_empty(n, _U8, logits, dev, stream))
    sc = 0 if scores is None else _flat(scores, rows, dev, _F32, "scores")
    ln = 0 if lengths is None else _flat(lengths, rows, dev, _I32, "lengths")
    fi = 0 if finished is None else _flat(finished, rows, dev, _U8, "finished")
    ho = 0 if hist_off is None else _flat(hist_off, rows + 1, dev, _I32, "hist_off")
    hi = 0 if hist_ids is None else _flat(hist_ids, 0, dev, _I32, "hist_ids") or ho     # (an empty tensor has no address)
    mk = mask_ld = 0
    mr = 0 if mask_row is None else _flat(mask_row, rows, dev, _I32, "mask_row")
    if mask is not None:
        m_rows, words, mask_ld = _rows2d(mask, dev, _I32, "mask")
        _want(words >= (V + 31) // 32 and (mr or m_rows >= rows), "mask: the words of every row are wanted")
        mk = mask.data_ptr()
    st = 0 if status is None else _flat(status, 1, dev, _I32, "status")
    to = (_flat(out["tokens"], n, dev, _I32, "tokens"), _flat(out["parents"], n, dev, _I32, "parents"),
          _flat(out["scores"], n, dev, _F32, "scores"), _flat(out["lengths"], n, dev, _I32, "lengths"),
          _flat(out["finished"], n, dev, _U8, "finished"))
    if groups:
        _call(dev, stream, "dlk_beam_select", _lib.lib().dlk_beam_select,
              _lib.BeamBatch(logits.data_ptr(), ld, ho, hi, mk, mask_ld, mr, sc, ln, fi, *to, st), groups, V,
              _lib.BeamParams(beams, n_out, eos_id, length_penalty, repeat_penalty, frequency_penalty,
                              presence_penalty, order, max_history))
    return out


def _span(sizes, strides) -> Optional[tuple]:
    """(count, stride) of several dimensions walked as one, or None where they are no single stride."""
    n, stride = 1, 0
    for size, st in zip(reversed(sizes), reversed(strides)):
        if size == 1:
            continue
        if n == 1:
            n, stride = size, st
        elif st == n * stride:
            n *= size
        else:
            return None
    return n, stride


def beam_state(src: torch.Tensor, dst: Optional[torch.Tensor] = None, row_dim: int = 0,
               length_dim: Optional[int] = None, length: Optional[int] = None) -> _lib.BeamState:
    """The rows (dimension row_dim) of a tensor as a state of beam_reorder, in place unless dst is given; only the
    first `length` entries of dimension length_dim where that is given (the filled part of a cache).  The
    dimensions before the rows, those up to length_dim and those from it on have to be one stride each.  The
    caller keeps the tensors."""
    size = src.shape
    nd = len(size)
    cut = row_dim + 1 if length_dim is None else length_dim
    if not (0 <= row_dim < nd and (length_dim is None or row_dim < cut < nd)):
        raise ValueError("length_dim: a dimension after the rows is wanted")
    if length is None or length_dim is None:
        length = size[cut] if cut < nd else 1
    elif not 0 <= length <= size[cut]:
        raise ValueError("length: more than the tensors hold")
    rows, item = size[row_dim], src.element_size()
    if dst is None and src.is_contiguous():
        # by the sizes: strides of single rows or heads may be anything
        outer = inner = 1
        for n in size[:row_dim]:
            outer *= n
        for n in size[row_dim + 1:cut]:
            inner *= n
        entry = item
        for n in size[cut + 1:]:
            entry *= n
        if (outer | inner) >> 31:
            raise ValueError(_WIDE.format("beam_state"))
        room = entry * size[cut] if cut < nd else entry
        row = room * inner
        at, dev = src.data_ptr(), src.get_device()
        s = _lib.BeamState(at, at, entry * length, row, row * rows, room, row, row * rows, room, outer, inner)
        s.rows = (rows, rows, dev, dev)
        return s
    shape = list(size)
    if length_dim is not None:
        shape[cut] = length
    dst_rows = rows
    if dst is not None:
        other = list(dst.shape)
        _want(len(other) == nd and dst.dtype == src.dtype, "dst: a tensor of src's kind is wanted")
        dst_rows = other[row_dim]
        other[row_dim] = rows
        if length_dim is not None and other[cut] >= shape[cut]:
            other[cut] = shape[cut]
        _want(other == shape, "dst: another shape than src's")

    def layout(t):
        st = t.stride()
        outer, inner = _span(shape[:row_dim], st[:row_dim]), _span(shape[row_dim + 1:cut], st[row_dim + 1:cut])
        rest = _span(shape[cut:], st[cut:])
        _want(outer is not None and inner is not None and rest is not None and (rest[0] == 1 or rest[1] == 1),
              "strides that are not one per part, or rows whose entries are apart")
        return t.data_ptr(), st[row_dim] * item, outer, inner, rest[0] * item
    at, row, outer, inner, width = layout(src)
    d_at, d_row, d_outer, d_inner, _ = (at, row, outer, inner, width) if dst is None else layout(dst)
    _want((outer[0] | inner[0]) >> 31 == 0, _WIDE.format("beam_state"))
    s = _lib.BeamState(at, d_at, 0 if 0 in shape else width, row, outer[1] * item, inner[1] * item, d_row,
                       d_outer[1] * item, d_inner[1] * item, outer[0], inner[0])
    s.rows = (rows, dst_rows, src.get_device(), src.get_device() if dst is None else dst.get_device())
    return s


def beam_history(off: torch.Tensor, ids: torch.Tensor, tokens: Optional[torch.Tensor], max_history: int,
                 out_off: torch.Tensor, out_ids: torch.Tensor) -> _lib.BeamHistory:
    """The rows' histories (CSR) and the tokens to append, for beam_reorder; out_ids has room for max_history ids
    of every new row.  The caller keeps the tensors."""
    if not -0x80000000 <= max_history <= 0x7fffffff:
        raise ValueError(_WIDE.format("beam_history"))
    dev = off.get_device()
    some = (off, ids, out_off, out_ids) if tokens is None else (off, ids, out_off, out_ids, tokens)
    for t in some:
        if t.dtype is not _I32 or t.get_device() != dev or not t.is_contiguous():
            raise ValueError("history: contiguous values of int32 on one device are wanted")
    at = off.data_ptr()
    h = _lib.BeamHistory(at, ids.data_ptr() or at, 0 if tokens is None else tokens.data_ptr(), max_history,
                         out_off.data_ptr(), out_ids.data_ptr())
    h.sizes = (off.numel(), None if tokens is None else tokens.numel(), out_off.numel(), out_ids.numel(), dev)
    return h


_STATES = {n: _lib.BeamState * n for n in range(1, 9)}


def beam_reorder(parents: torch.Tensor, beams: int, n_out: int, states=(), history: Optional[_lib.BeamHistory] = None,
                 stream: Optional[int] = None) -> None:
    """The states (beam_state) and histories (beam_history) of the new rows from their parents' (dlk_beam_reorder);
    parents int32 [groups * n_out] as beam_select writes them."""
    dev = parents.get_device()
    at = _flat(parents, 0, dev, _I32, "parents")
    total = parents.numel()
    _want(beams > 0 and n_out > 0 and total % n_out == 0, "parents: whole groups of n_out are wanted")
    groups = total // n_out
    if (beams | n_out | groups) >> 31:
        raise ValueError(_WIDE.format("beam_reorder"))
    for s in states:
        _want(s.rows[0] >= groups * beams and s.rows[1] >= total, "states: fewer rows than the groups have")
        _want(s.rows[2] == dev and s.rows[3] == dev, "states: tensors on the call's device are wanted")
    if history is not None:
        n_off, n_tok, n_out_off, n_out_ids, where = history.sizes
        _want(n_off >= groups * beams + 1 and n_out_off >= total + 1 and (n_tok is None or n_tok >= total) and
              n_out_ids >= total * history.max_history, "history: fewer entries than the groups need")
        _want(where == dev, "history: tensors on the call's device are wanted")
    if groups:
        k = len(states)
        arr = (_STATES.get(k) or _lib.BeamState * k)(*states) if k else None
        _call(dev, stream, "dlk_beam_reorder", _lib.lib().dlk_beam_reorder, at, groups, beams, n_out, arr, k, history)
