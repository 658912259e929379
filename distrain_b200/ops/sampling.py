"""Logits of the serving path before a token is drawn: penalties for repeated tokens, biases, token masks."""
from __future__ import annotations

import struct

import torch

from .paged import _F32, _I32, _fail, _launch, _stream, _vec, on_current_device

MAX_BIAS = 16384
_LOGITS = struct.Struct("=12Q5q6i").pack  # argument struct of the launcher (csrc/kernels/logits.cu)


def _matrix(name, t, rows, cols, dtype):
    if t.dtype != dtype or t.dim() != 2 or t.shape[0] != rows or (cols is not None and t.shape[1] != cols) or \
            (t.shape[1] > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < 0):
        _fail(f"{name}: expected {dtype} [{rows}, {'columns' if cols is None else cols}] with unit column stride, got "
              f"{t.dtype} {tuple(t.shape)} strides {t.stride()}")


def process_logits(logits, out, *, history=None, lens=None, prompt_lens=None, repetition=None, presence=None,
                   frequency=None, bias_ids=None, bias_vals=None, bias_lens=None, mask=None, stream=None):
    """``out`` [B, V] fp32 from ``logits`` [B, V] (fp32 or bf16; rows may be strided; fp32 ``out`` may be ``logits``,
    and shares memory with no input otherwise).

    With c = how often token v occurs in ``history[b, prompt_lens[b]:lens[b]]`` (the answer so far; the whole
    row without ``prompt_lens``) and *seen* = it occurs in ``history[b, :lens[b]]``, in this order:

        seen:  z = z / repetition[b] if z > 0 else z * repetition[b]
        c > 0: z = z - frequency[b] * c - presence[b]
        z = z + the sum of ``bias_vals[b, e]`` with ``bias_ids[b, e]`` = v, e < ``bias_lens[b]``
        z = -inf where bit v % 32 of ``mask[b, v // 32]`` is 0 (whatever z was)

    ``history`` int32 [B, L] with ``lens`` int32 [B] (beyond L: L); ids outside [0, V) are ignored there and in
    ``bias_ids`` (at most ``MAX_BIAS`` entries a row). ``repetition`` (positive) / ``presence`` / ``frequency`` finite
    fp32 [B], 1 / 0 / 0 when None. ``mask`` int32
    [B, ceil(V / 32)] (one row expanded to B works). A row whose mask has no bit set is all -inf."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        _fail(f"logits: fp32 or bf16 [B, V], got {logits.dtype} {tuple(logits.shape)}")
    B, V = logits.shape
    if V < 1 or V >= 1 << 30 or B > 65535:
        _fail(f"logits: 1 <= V < 2^30 and B <= 65535, got {B} x {V}")
    ldx = ldo = V
    if not (out.shape == (B, V) and out.dtype is _F32 and logits.is_contiguous() and out.is_contiguous()):
        _matrix("logits", logits, B, V, logits.dtype)
        _matrix("out", out, B, V, torch.float32)
        if B > 1:
            ldx, ldo = logits.stride(0), out.stride(0)
        if ldo < V:
            _fail("out: rows overlap")
    xp, op = logits.data_ptr(), out.data_ptr()
    if op == xp and (logits.dtype != torch.float32 or ldx != ldo):
        _fail("out may be logits only for fp32 logits of the same strides")
    L = K = ldh = ldb = ldm = hp = np = pp = rp = ap = fp = ip = vp = cp = mp = 0
    if history is not None:
        if lens is None:
            _fail("history needs lens")
        _matrix("history", history, B, None, torch.int32)
        _vec("lens", lens, B)
        if prompt_lens is not None:
            _vec("prompt_lens", prompt_lens, B)
            np = prompt_lens.data_ptr()
        L, ldh = history.shape[1], history.stride(0)
        if L >= 1 << 23:
            _fail("history: below 2^23 tokens a row")
        hp, pp = history.data_ptr(), lens.data_ptr()
        if repetition is not None:
            _vec("repetition", repetition, B, _F32)
            rp = repetition.data_ptr()
        if presence is not None:
            _vec("presence", presence, B, _F32)
            ap = presence.data_ptr()
        if frequency is not None:
            _vec("frequency", frequency, B, _F32)
            fp = frequency.data_ptr()
    elif lens is not None or prompt_lens is not None or repetition is not None or presence is not None or \
            frequency is not None:
        _fail("penalties need history and lens")
    if bias_ids is not None or bias_vals is not None or bias_lens is not None:
        if bias_ids is None or bias_vals is None or bias_lens is None:
            _fail("biases need bias_ids, bias_vals and bias_lens")
        _matrix("bias_ids", bias_ids, B, None, torch.int32)
        K = bias_ids.shape[1]
        _matrix("bias_vals", bias_vals, B, K, torch.float32)
        _vec("bias_lens", bias_lens, B)
        ldb = bias_ids.stride(0)
        if K > MAX_BIAS:
            _fail(f"bias_ids: at most {MAX_BIAS} entries a row")
        if B > 1 and bias_vals.stride(0) != ldb:
            _fail("bias_ids and bias_vals: the same row stride")
        ip, vp, cp = bias_ids.data_ptr(), bias_vals.data_ptr(), bias_lens.data_ptr()
    if mask is not None:
        _matrix("mask", mask, B, (V + 31) // 32, torch.int32)
        ldm, mp = mask.stride(0), mask.data_ptr()
    dev = on_current_device(logits, out, history, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias_vals,
                            bias_lens, mask)
    if B == 0:
        return
    _launch("dt_process_logits", _LOGITS(xp, op, hp, np, pp, rp, ap, fp, ip, vp, cp, mp, ldx, ldo, ldh, ldb, ldm,
                                         logits.dtype is torch.bfloat16, B, V, L, K, 0), _stream(stream, dev))
