"""Log probabilities of given classes, with the entropy and the top alternatives (y3_log_probs, include/yolo3hip.h).

    log_probs(logits, ids, top=5) -> ClassProbs(logp, entropy, top_ids, top_logp)

For a detector's head the class logits of a box that holds one object: independent sigmoids p_c of which exactly one is on
give P(c) proportional to p_c / (1 - p_c) = exp(z_c), the softmax of the logits whose sigmoids the decode takes
(utils/utils.py:90-96).  `inference.alternatives` does it for the boxes NMS kept.
"""
import collections
import ctypes

import torch

from . import _lib
from .linear_i8 import _forward_ad, _refuse_gradient, _stream_of

MAX_TOP, MAX_CLASSES = 32, 1 << 24      # what the library takes; its own check sees 32 bits of a size only
ClassProbs = collections.namedtuple("ClassProbs", "logp entropy top_ids top_logp")
_DESCS = {}


def _two_strides(t):
    """(rows, group, group_ld, row_ld) of a tensor [..., C] whose leading dimensions are at most two uniform strides, else
    None."""
    dims = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    merged = []
    for n, s in reversed(dims):                     # innermost first
        if merged and s == merged[-1][0] * merged[-1][1]:
            merged[-1] = (merged[-1][0] * n, merged[-1][1])
        else:
            merged.append((n, s))
    if not merged:
        return 1, 1, 0, 0
    if len(merged) == 1:
        return merged[0][0], 1, merged[0][1], 0
    if len(merged) == 2 and merged[0][0] < 1 << 31:        # (a group is a 32-bit number)
        return merged[0][0] * merged[1][0], merged[0][0], merged[1][1], merged[0][1]
    return None


def _descriptor(key):
    hit = _DESCS.get(key)
    if hit is None:
        d = _lib.LogProbsDesc()
        d.dtype, d.classes, d.rows, d.group, d.group_ld, d.row_ld, d.top, d.ids_64, d.extent = key
        need = ctypes.c_int64(0)
        _lib.check(_lib.load().y3_log_probs_workspace_bytes(ctypes.byref(d), ctypes.byref(need)))
        if len(_DESCS) >= 256:
            _DESCS.clear()
        hit = _DESCS[key] = (ctypes.byref(d), int(need.value))
    return hit


def log_probs(logits, ids=None, top=0, rows=None, classes=None, out=None):
    """logits [..., C] float32 / bfloat16; ids [...] int32 / int64: the class whose log probability is wanted (negative:
    none, logp 0); top: how many alternatives (0 .. 32).  Returns ClassProbs: logp [...] (None without ids), entropy [...],
    top_ids int32 [..., top] and top_logp [..., top] (None with top = 0), largest first, ties to the lowest class.
    -inf logits are impossible classes; a row of nothing else has log p -inf and entropy 0; a NaN or +inf makes a row NaN.

    rows: int64 [R] element offsets into a contiguous `logits` of any shape at which rows of `classes` logits start; a
    negative one is skipped: its outputs stay what `out` holds (without `out`: zeros, class -1).  An offset whose row would
    end behind the tensor gives NaN and class -1.
    out: (logp, entropy, top_ids, top_logp) to write into, contiguous; None where there is no such output."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a tensor on the GPU")
    forward = _forward_ad._current_level >= 0
    if forward or logits.requires_grad:
        _refuse_gradient(logits, "logits", "log_probs")
    if logits.dtype == torch.float32:
        code = _lib.Y3_F32
    elif logits.dtype == torch.bfloat16:
        code = _lib.Y3_BF16
    else:
        raise ValueError("logits must be float32 or bfloat16, got %s" % logits.dtype)
    top, device = int(top), logits.device
    if device.index != torch.cuda.current_device():             # launches go to the current device
        with torch.cuda.device(device):
            return log_probs(logits, ids, top=top, rows=rows, classes=classes, out=out)
    if rows is None:
        if classes is not None:
            raise ValueError("classes goes with rows")
        if logits.dim() < 1 or logits.shape[-1] < 1:
            raise ValueError("logits must be [..., C], got %r" % (tuple(logits.shape),))
        C, lead = logits.shape[-1], logits.shape[:-1]
        if C > MAX_CLASSES:
            raise ValueError("%d classes, at most %d" % (C, MAX_CLASSES))
        if len(lead) == 1 and (C == 1 or logits.stride(1) == 1):
            n, group, group_ld, row_ld = lead[0], 1, logits.stride(0), 0
        else:
            strides = _two_strides(logits) if C == 1 or logits.stride(-1) == 1 else None
            if strides is None:
                logits = logits.contiguous()
                strides = _two_strides(logits)
            n, group, group_ld, row_ld = strides
            if 0 in lead:
                n, group = 0, 1
        extent, rows_ptr = 1 << 42, None
    else:
        if classes is None or not 1 <= int(classes) <= MAX_CLASSES:
            raise ValueError("rows needs classes, 1 .. %d" % MAX_CLASSES)
        if rows.dtype != torch.int64 or rows.dim() != 1 or rows.device != device:
            raise ValueError("rows must be int64 [R] on %s" % device)
        if not logits.is_contiguous():
            raise ValueError("rows are offsets into contiguous logits")
        rows = rows.contiguous()
        C, lead, n = int(classes), rows.shape, rows.shape[0]
        group, group_ld, row_ld, extent, rows_ptr = 1, 0, 0, logits.numel(), rows.data_ptr()
    if not 0 <= top <= min(MAX_TOP, C):
        raise ValueError("top = %d: 0 .. %d of %d classes" % (top, min(MAX_TOP, C), C))
    ids_ptr, ids_64 = None, 0
    if ids is not None:
        if ids.dtype not in (torch.int32, torch.int64) or ids.shape != lead or ids.device != device:
            raise ValueError("ids must be int32 or int64 %r on %s" % (tuple(lead), device))
        ids = ids.contiguous()
        ids_ptr, ids_64 = ids.data_ptr(), int(ids.dtype == torch.int64)
    if out is None:
        if rows is None:
            entropy = logits.new_empty(lead, dtype=torch.float32)
            logp = torch.empty_like(entropy) if ids is not None else None
            top_logp = logits.new_empty(lead + (top,), dtype=torch.float32) if top else None
            top_ids = torch.empty_like(top_logp, dtype=torch.int32) if top else None
        else:
            logp = torch.zeros(lead, dtype=torch.float32, device=device) if ids is not None else None
            entropy = torch.zeros(lead, dtype=torch.float32, device=device)
            top_ids = torch.full(lead + (top,), -1, dtype=torch.int32, device=device) if top else None
            top_logp = torch.zeros(lead + (top,), dtype=torch.float32, device=device) if top else None
    else:
        logp, entropy, top_ids, top_logp = out
        for t, shape, dtype, want in ((logp, lead, torch.float32, ids is not None), (entropy, lead, torch.float32, None),
                                      (top_ids, lead + (top,), torch.int32, top > 0), (top_logp, lead + (top,), torch.float32, top > 0)):
            if want is not None and (t is not None) != want:
                raise ValueError("out: logp goes with ids, top_ids and top_logp with top")
            if t is not None and (t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous()):
                raise ValueError("out: expected contiguous %s %r on %s" % (dtype, tuple(shape), device))
            if t is not None and (forward or t.requires_grad):
                _refuse_gradient(t, "out", "log_probs")
    if n and (ids is not None or top or entropy is not None):
        dref, need = _descriptor((code, C, n, group, group_ld, row_ld, top, ids_64, extent))
        ws = logits.new_empty(need, dtype=torch.uint8) if need else None
        rc = _lib.load().y3_log_probs(dref, logits.data_ptr(), rows_ptr, ids_ptr,
                                      logp.data_ptr() if logp is not None else None,
                                      entropy.data_ptr() if entropy is not None else None,
                                      top_ids.data_ptr() if top else None, top_logp.data_ptr() if top else None,
                                      ws.data_ptr() if need else None, need, _stream_of(device.index))
        if rc:
            _lib.check(rc)
    return ClassProbs(logp, entropy, top_ids, top_logp)
