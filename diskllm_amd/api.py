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
# Tensors on one device, the call on that device's current stream unless `stream` says
# otherwise; what does not fit raises ValueError before anything is launched.

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on(device, *tensors) -> None:
    for t in tensors:
        _want(t is None or t.device == device, "tensors on different devices")


def _rows2d(t: torch.Tensor, what: str) -> int:
    """The row stride of a [rows, n] tensor whose rows are contiguous."""
    _want(t.dim() == 2 and (t.shape[1] == 1 or t.stride(1) == 1), f"{what}: [rows, n] with contiguous rows is wanted")
    ld = t.stride(0)
    if t.shape[0] <= 1:
        return max(ld, t.shape[1])
    _want(ld >= t.shape[1], f"{what}: rows overlap")
    return ld


def _flat(t: Optional[torch.Tensor], n: int, dtype, what: str) -> None:
    _want(t is None or (t.numel() >= n and t.dtype == dtype and t.is_contiguous()),
          f"{what}: at least {n} contiguous values of {dtype} are wanted")


def _call(device, stream, what: str, fn, *args) -> None:
    """fn(*args, stream) with `device` current (the kernels run there)."""
    _want(device.type == "cuda", f"{what}: tensors on the GPU are wanted")
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream if stream is not None else torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream if stream is not None else torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        _lib.check(rc, what)


def quantize_rows(x: torch.Tensor, q: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                  stream: Optional[int] = None):
    """(q int8 [rows, n], scale float32 [rows]) of x [rows, n] in float32, bfloat16 or float16: hidden states with a
    scale per token, or weights [vocab, n] with one per channel (dlk_quantize_rows)."""
    _want(x.dtype in _DTYPES, "x: float32, bfloat16 or float16 is wanted")
    ldx = _rows2d(x, "x")
    rows, n = x.shape
    if q is None:
        q = torch.empty((rows, (n + 15) // 16 * 16), dtype=torch.int8, device=x.device)[:, :n]
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    ldq = _rows2d(q, "q")
    _want(q.shape == x.shape and q.dtype == torch.int8, "q: int8 of x's shape is wanted")
    _flat(scale, rows, torch.float32, "scale")
    _on(x.device, q, scale)
    if rows == 0:
        return q, scale
    _call(x.device, stream, "dlk_quantize_rows", _lib.lib().dlk_quantize_rows, x.data_ptr(), _DTYPES[x.dtype], ldx,
          rows, n, q.data_ptr(), ldq, scale.data_ptr())
    return q, scale


def logits_i8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, softcap: float = 0.0,
              out: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """Logits float32 [rows, vocab] of x int8 [rows, n] (x_scale [rows]) over w int8 [vocab, n] (w_scale [vocab]),
    soft-capped where softcap > 0 (dlk_logits_i8)."""
    _want(x.dtype == torch.int8 and w.dtype == torch.int8, "x and w: int8 is wanted")
    ldx, ldw = _rows2d(x, "x"), _rows2d(w, "w")
    rows, n = x.shape
    V = w.shape[0]
    _want(w.shape[1] == n, "x and w: rows of one length are wanted")
    if out is None:
        out = torch.empty((rows, (V + 63) // 64 * 64), dtype=torch.float32, device=x.device)[:, :V]
    ld = _rows2d(out, "out")
    _want(out.shape == (rows, V) and out.dtype == torch.float32, "out: float32 [rows, vocab] is wanted")
    _flat(x_scale, rows, torch.float32, "x_scale")
    _flat(w_scale, V, torch.float32, "w_scale")
    _on(x.device, x_scale, w, w_scale, out)
    if rows == 0:
        return out
    _call(x.device, stream, "dlk_logits_i8", _lib.lib().dlk_logits_i8, x.data_ptr(), ldx, x_scale.data_ptr(),
          w.data_ptr(), ldw, w_scale.data_ptr(), rows, V, n, float(softcap), out.data_ptr(), ld)
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
    _want(logits.dtype == torch.float32, "logits: float32 is wanted")
    ld = _rows2d(logits, "logits")
    rows, V = logits.shape
    _want(beams > 0 and n_out > 0 and rows % beams == 0, "logits: whole groups of beams are wanted")
    groups = rows // beams
    dev = logits.device
    if out is None:
        out = dict(tokens=torch.empty(groups * n_out, dtype=torch.int32, device=dev),
                   parents=torch.empty(groups * n_out, dtype=torch.int32, device=dev),
                   scores=torch.empty(groups * n_out, dtype=torch.float32, device=dev),
                   lengths=torch.empty(groups * n_out, dtype=torch.int32, device=dev),
                   finished=torch.empty(groups * n_out, dtype=torch.uint8, device=dev))
    for k, t, n, dt in (("scores", scores, rows, torch.float32), ("lengths", lengths, rows, torch.int32),
                        ("finished", finished, rows, torch.uint8), ("hist_off", hist_off, rows + 1, torch.int32),
                        ("hist_ids", hist_ids, 0, torch.int32), ("mask_row", mask_row, rows, torch.int32),
                        ("status", status, 1, torch.int32)):
        if t is not None:
            _flat(t, n, dt, k)
            _want(t.device == dev, "tensors on different devices")
    mask_ld = 0
    if mask is not None:
        mask_ld = _rows2d(mask, "mask")
        _want(mask.dtype == torch.int32 and mask.shape[1] >= (V + 31) // 32 and mask.device == dev and
              (mask_row is not None or mask.shape[0] >= rows), "mask: int32 words of every row are wanted")
    for k, dt in (("tokens", torch.int32), ("parents", torch.int32), ("scores", torch.float32),
                  ("lengths", torch.int32), ("finished", torch.uint8)):
        _flat(out[k], groups * n_out, dt, k)
        _want(out[k].device == dev, "tensors on different devices")
    if groups == 0:
        return out
    b = _lib.BeamBatch(
        logits=logits.data_ptr(), ld=ld, hist_off=_ptr(hist_off),
        hist_ids=_ptr(hist_ids) or _ptr(hist_off) if hist_ids is not None else None,   # (an empty tensor has no address)
        mask=_ptr(mask), mask_ld=mask_ld, mask_row=_ptr(mask_row), scores=_ptr(scores), lengths=_ptr(lengths), finished=_ptr(finished),
        out_tokens=out["tokens"].data_ptr(), out_parents=out["parents"].data_ptr(),
        out_scores=out["scores"].data_ptr(), out_lengths=out["lengths"].data_ptr(),
        out_finished=out["finished"].data_ptr(), status=_ptr(status))
    p = _lib.BeamParams(beams, n_out, eos_id, length_penalty, repeat_penalty, frequency_penalty, presence_penalty,
                        order, max_history)
    _call(dev, stream, "dlk_beam_select", _lib.lib().dlk_beam_select, C.byref(b), groups, V, C.byref(p))
    return out


def _span(sizes, strides) -> Optional[tuple]:
    """(count, stride) of several dimensions walked as one, or None where they are no single stride."""
    n, stride = 1, 0
    for size, st in reversed(list(zip(sizes, strides))):
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
    dst = src if dst is None else dst
    nd = src.dim()
    _want(0 <= row_dim < nd and dst.dim() == nd and dst.dtype == src.dtype, "dst: a tensor of src's kind is wanted")
    cut = row_dim + 1 if length_dim is None else length_dim
    _want(row_dim < cut < nd or length_dim is None, "length_dim: a dimension after the rows is wanted")
    shape = list(src.shape)
    if length_dim is not None and length is not None:
        _want(0 <= length <= min(src.shape[length_dim], dst.shape[length_dim]), "length: more than the tensors hold")
        shape[length_dim] = length
    _want(all(a == b for i, (a, b) in enumerate(zip(src.shape, dst.shape)) if i not in (row_dim, length_dim)) and
          (length_dim is None or shape[length_dim] <= dst.shape[length_dim]), "dst: another shape than src's")
    item = src.element_size()
    s = _lib.BeamState()
    for t, k in ((src, "src"), (dst, "dst")):
        outer = _span(shape[:row_dim], t.stride()[:row_dim])
        inner = _span(shape[row_dim + 1:cut], t.stride()[row_dim + 1:cut])
        rest = _span(shape[cut:], t.stride()[cut:])
        _want(None not in (outer, inner, rest) and (rest[0] == 1 or rest[1] == 1),
              f"{k}: strides that are not one per part, or rows whose entries are apart")
        setattr(s, k, t.data_ptr())
        setattr(s, k + "_row", t.stride(row_dim) * item)
        setattr(s, k + "_outer", outer[1] * item)
        setattr(s, k + "_inner", inner[1] * item)
        s.n_outer, s.n_inner, s.bytes = outer[0], inner[0], rest[0] * item
    if 0 in shape:
        s.bytes = 0
    s.rows = (src.shape[row_dim], dst.shape[row_dim], src.device, dst.device)
    return s


def beam_history(off: torch.Tensor, ids: torch.Tensor, tokens: Optional[torch.Tensor], max_history: int,
                 out_off: torch.Tensor, out_ids: torch.Tensor) -> _lib.BeamHistory:
    """The rows' histories (CSR) and the tokens to append, for beam_reorder; out_ids has room for max_history ids
    of every new row.  The caller keeps the tensors."""
    for k, t in (("off", off), ("ids", ids), ("tokens", tokens), ("out_off", out_off), ("out_ids", out_ids)):
        _flat(t, 0, torch.int32, k)
        _want(t is None or t.device == off.device, "tensors on different devices")
    h = _lib.BeamHistory(off.data_ptr(), ids.data_ptr() or off.data_ptr(), _ptr(tokens), max_history, out_off.data_ptr(),
                         out_ids.data_ptr())
    h.sizes = (off.numel(), None if tokens is None else tokens.numel(), out_off.numel(), out_ids.numel(), off.device)
    return h


def beam_reorder(parents: torch.Tensor, beams: int, n_out: int, states=(), history: Optional[_lib.BeamHistory] = None,
                 stream: Optional[int] = None) -> None:
    """The states (beam_state) and histories (beam_history) of the new rows from their parents' (dlk_beam_reorder);
    parents int32 [groups * n_out] as beam_select writes them."""
    _flat(parents, 0, torch.int32, "parents")
    _want(beams > 0 and n_out > 0 and parents.numel() % n_out == 0, "parents: whole groups of n_out are wanted")
    groups = parents.numel() // n_out
    dev = parents.device
    for s in states:
        _want(s.rows[0] >= groups * beams and s.rows[1] >= groups * n_out, "states: fewer rows than the groups have")
        _want(s.rows[2] == dev and s.rows[3] == dev, "tensors on different devices")
    if history is not None:
        n_off, n_tok, n_out_off, n_out_ids, where = history.sizes
        _want(n_off >= groups * beams + 1 and n_out_off >= groups * n_out + 1 and
              (n_tok is None or n_tok >= groups * n_out) and
              n_out_ids >= groups * n_out * history.max_history, "history: fewer entries than the groups need")
        _want(where == dev, "tensors on different devices")
    if groups == 0:
        return
    arr = (_lib.BeamState * max(len(states), 1))(*states)
    _call(dev, stream, "dlk_beam_reorder", _lib.lib().dlk_beam_reorder, parents.data_ptr(), groups, beams, n_out, arr,
          len(states), C.byref(history) if history is not None else None)
