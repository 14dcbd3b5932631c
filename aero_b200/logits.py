"""Logits of a batch adjusted before sampling (aero_cuda_logits_adjust,
include/aero_cuda_pages.h): penalties for repeated tokens, biases, grammar masks; and
tokens drawn from them (aero_cuda_logits_sample): temperature, top-k, top-p, min-p.
"""

from __future__ import annotations

from . import native_cuda as nc

_KINDS = None  # torch types -> element types
_TORCH = None  # torch, float32, int32


def _kinds():
    global _KINDS, _TORCH
    if _KINDS is None:
        import torch
        nc.require_gpu()
        _TORCH = torch, torch.float32, torch.int32
        _KINDS = {torch.float32: nc.TYPE_F32, torch.float16: nc.TYPE_F16, torch.bfloat16: nc.TYPE_BF16}
    return _KINDS


def adjust(logits, *, history=None, n_history=None, n_prompt=None, repetition=None, frequency=None, presence=None,
           bias_start=None, bias_token=None, bias_value=None, mask=None, out=None):
    """logits (rows, vocab), a CUDA tensor of float32, float16 or bfloat16; returns out (a new
    tensor, or the one given: it may be logits itself).

    history (rows, length) int32 token ids, the first n_history[r] of row r counted (at most
    length), of which the first n_prompt[r] are the prompt (the repetition penalty takes all of
    them, the others what follows the prompt). History and mask may be views: slices of wider
    tensors, or one row expanded over all. repetition, frequency, presence: float32 (rows).
    Biases: row r's entries are [bias_start[r], bias_start[r + 1]) of bias_token (int32)
    and bias_value (float32); what these name outside the two is passed over. mask: int32
    (rows, at least (vocab + 31) // 32), bit token % 32 of word token // 32 set where the token
    is allowed. Runs on torch's current stream."""
    import torch
    L, kinds = nc.lib(), _kinds()
    f32, i32 = torch.float32, torch.int32
    index = logits.get_device()
    if logits.dim() != 2 or logits.dtype not in kinds or index < 0 or logits.stride(1) != 1:
        raise ValueError("logits must be a (rows, vocab) CUDA tensor of float32, float16 or bfloat16, contiguous along vocab")
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((rows, vocab))
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.get_device() != index or out.stride(1) != 1:
        raise ValueError("out must have the logits' shape, type and device")

    def vec(t, name, dtype, n):
        if t is None:
            return None
        if t.dtype is not dtype or t.get_device() != index or (n >= 0 and t.numel() != n) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dtype}" + (f", {n} entries," if n >= 0 else "") + f" on {logits.device}")
        return t.data_ptr()

    def mat(t, name, width):
        if t is None:
            return None, 0, 0
        shape = t.shape
        if t.dtype is not i32 or t.get_device() != index or len(shape) != 2 or shape[0] != rows or shape[1] < width:
            raise ValueError(f"{name} must be int32 ({rows}, at least {width}) on {logits.device}")
        stride, one = t.stride()
        if one != 1 and shape[1] > 1:
            raise ValueError(f"{name} must be contiguous along its rows")
        return t.data_ptr(), stride if rows > 1 else shape[1], shape[1]

    if (history is None) != (n_history is None):
        raise ValueError("history and n_history come together")
    if (bias_start is None) != (bias_token is None) or (bias_start is None) != (bias_value is None):
        raise ValueError("bias_start, bias_token and bias_value come together")
    if bias_token is not None:
        if bias_token.numel() != bias_value.numel():
            raise ValueError("bias_token and bias_value differ in length")
        if bias_token.numel() == 0:
            bias_start = bias_token = bias_value = None
    if history is not None and history.shape[-1] == 0:
        history = n_history = None
    hp, hl, hw = mat(history, "history", 0)
    mp, mlw, _ = mat(mask, "mask", (vocab + 31) // 32)
    if L.aero_cuda_logits_adjust_views(
            logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, kinds[logits.dtype], rows, vocab, hp, hl, hw,
            vec(n_history, "n_history", i32, rows), vec(n_prompt, "n_prompt", i32, rows),
            vec(repetition, "repetition", f32, rows), vec(frequency, "frequency", f32, rows),
            vec(presence, "presence", f32, rows), vec(bias_start, "bias_start", i32, rows + 1),
            vec(bias_token, "bias_token", i32, -1), vec(bias_value, "bias_value", f32, -1),
            0 if bias_token is None else bias_token.numel(), mp, mlw, out.data_ptr(),
            out.stride(0) if rows > 1 else vocab, torch._C._cuda_getCurrentRawStream(index) or None) != 0:
        raise ValueError(f"logits_adjust refused: {nc.last_error()}")
    return out


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, logprob=False, out=None):
    """A token from each row of logits (rows, vocab), a CUDA tensor of float32, float16 or bfloat16, with the
    random numbers u (rows) float32 in [0, 1): int32 (rows), a new tensor or `out`; with logprob also the logs of the
    probabilities they were drawn with, float32 (rows).

    In falling order of the logits (equal ones: the lower token) with weights exp((x - largest) / temperature), kept are the
    first top_k; of those the ones up to where the running sum reaches top_p of the whole; of those the ones with
    at least min_p of the largest weight. Drawn is the first whose running sum exceeds u times the sum of the kept.
    temperature, top_p, min_p: float32 (rows), top_k: int32 (rows); None, or a row's top_k of 0 or less, top_p of 1 or
    more, min_p of 0 or less: no such limit; a row's temperature of 0 or less: the largest logit. Logits of -infinity and
    those that are no number are never drawn; -1 for a row of nothing else. Runs on torch's current stream."""
    L, kinds = nc.lib(), _kinds()
    index, shape, kind = logits.get_device(), logits.shape, kinds.get(logits.dtype)
    if len(shape) != 2 or kind is None or index < 0 or logits.stride(1) != 1:
        raise ValueError("logits must be a (rows, vocab) CUDA tensor of float32, float16 or bfloat16, contiguous along vocab")
    rows, vocab = shape
    torch, f32, i32 = _TORCH

    def vec(t, name, dtype):
        if t.dtype is not dtype or t.get_device() != index or t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dtype}, {rows} entries, on {logits.device}")
        return t.data_ptr()

    if u is None:
        raise ValueError("u is required")
    if out is None:
        out = torch.empty(rows, dtype=i32, device=logits.device)
    logs = torch.empty(rows, dtype=f32, device=logits.device) if logprob else None
    if L.aero_cuda_logits_sample(
            logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, kind, rows, vocab, vec(u, "u", f32),
            None if temperature is None else vec(temperature, "temperature", f32),
            None if top_k is None else vec(top_k, "top_k", i32), None if top_p is None else vec(top_p, "top_p", f32),
            None if min_p is None else vec(min_p, "min_p", f32), vec(out, "out", i32),
            None if logs is None else logs.data_ptr(), torch._C._cuda_getCurrentRawStream(index) or None) != 0:
        raise ValueError(f"logits_sample refused: {nc.last_error()}")
    return (out, logs) if logprob else out
