"""Log probabilities of given tokens, with each row's entropy and top alternatives (``csrc/logprob.cu``, ``csrc/score_head.cu``).

A row's logits z, its token t, S = sum exp(z - max z):

    log p(t) = z_t - max z - ln S        H = - sum p ln p        the ``top`` largest z, of equal ones the lower id first

``token_logprobs`` takes logits that are there (a decode or verify step's, ``Engine.logits``); ``score`` and ``score_i8`` take rows
behind the final norm and the lm_head, and store no logits, or with alternatives those of a slab of rows at a time.  All sums are fp32.

A token outside the vocabulary (-1: no token) has log probability NaN; its row's other results are as ever.  A row without a finite
logit (every id banned) has log probabilities of -inf and entropy 0.  A NaN or +inf among a row's logits makes its numbers NaN.
Alternatives beyond the vocabulary have id -1 and log probability -inf.
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass
from typing import Optional

import torch

from . import lib as K

MAX_TOP = 32           # alternatives a row can have
SLAB_ELEMS = 160 << 20 # logits that ``score`` with alternatives keeps at a time (fewer where there is no room for them)
SLAB_ROWS = 32768      # rows whose sums it keeps at a time
MAX_I8_COLUMNS = 1 << 17


@dataclass(frozen=True)
class Logprobs:
    """Results of ``m`` rows: ``logprob``, ``entropy`` fp32 ``[m]``; ``top_ids`` int32 and ``top_logprobs`` fp32 ``[m][top]``, contiguous, on
    one device."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor

    def __post_init__(self):
        m, n, dev = self.logprob.shape[0], self.top_ids.shape[-1], self.logprob.device
        if n > MAX_TOP:
            raise ValueError(f"log probabilities of at most {MAX_TOP} alternatives, not {n}")
        for t, shape, dtype in ((self.logprob, (m,), torch.float32), (self.entropy, (m,), torch.float32), (self.top_ids, (m, n), torch.int32),
                                (self.top_logprobs, (m, n), torch.float32)):
            if t.shape != shape or t.dtype != dtype or t.device != dev or not t.is_contiguous():
                raise ValueError(f"results of {m} rows and {n} alternatives are contiguous fp32 / int32 tensors of {dev}")

    @staticmethod
    def empty(m: int, top: int, device) -> "Logprobs":
        if not 0 <= top <= MAX_TOP:
            raise ValueError(f"log probabilities of at most {MAX_TOP} alternatives, not {top}")
        f = lambda *s: torch.empty(s, dtype=torch.float32, device=device)           # noqa: E731
        return Logprobs._of(f(m), f(m), torch.empty((m, top), dtype=torch.int32, device=device), f(m, top))

    def rows(self, begin: int, end: int) -> "Logprobs":
        return Logprobs._of(self.logprob[begin:end], self.entropy[begin:end], self.top_ids[begin:end], self.top_logprobs[begin:end])

    @staticmethod
    def _of(logprob, entropy, top_ids, top_logprobs) -> "Logprobs":
        """Tensors that need no check."""
        out = object.__new__(Logprobs)
        out.__dict__.update(logprob=logprob, entropy=entropy, top_ids=top_ids, top_logprobs=top_logprobs)
        return out


def _results(m: int, top: Optional[int], out: Optional[Logprobs], device) -> Logprobs:
    if out is None:
        return Logprobs.empty(m, top or 0, device)
    got = out.top_ids.shape
    if got[0] != m or top is not None and top != got[1] or out.logprob.device != device:
        raise ValueError(f"results of {got[0]} rows and {got[1]} alternatives on {out.logprob.device}: {m} and {top} asked on {device}")
    return out


def _check_tokens(tokens: torch.Tensor, m: int, device):
    if tokens.dtype is not torch.int32 or tokens.shape != (m,) or tokens.device != device or m > 1 and tokens.stride(0) != 1:
        raise ValueError(f"tokens: {m} contiguous int32 ids on {device}")


def _rows_of(t: torch.Tensor, dtype, what: str, align: int = 4) -> tuple:
    """(rows, columns, elements from row to row, address) of a matrix."""
    shape = t.shape
    if len(shape) != 2 or t.dtype is not dtype or not t.is_cuda:
        raise ValueError(f"{what}: rows of {dtype} on a CUDA device")
    (m, n), (ld, step), at = shape, t.stride(), t.data_ptr()
    if n > 1 and step != 1:
        raise ValueError(f"{what}: one element after another")
    if m < 2:
        ld = (n + 15) // 16 * 16      # (a lone row's stride says nothing: a multiple of 16 bytes that holds it)
    elif ld < n:
        raise ValueError(f"{what}: rows that do not overlap")
    if at % align or ld * dtype.itemsize % align:
        raise ValueError(f"{what}: rows begin at multiples of {align} bytes")
    return m, n, ld, at


@functools.lru_cache(maxsize=None)
def _entry(name: str, kinds: str, result=ctypes.c_int):
    """An entry point of the library with its argument types (p: pointer, l: 64 bits, i: 32 bits), so that a call of a few microseconds
    wraps no numbers one by one."""
    fn = getattr(K.lib(), name)
    fn.restype = result
    fn.argtypes = [{"p": ctypes.c_void_p, "l": ctypes.c_longlong, "i": ctypes.c_int}[c] for c in kinds]
    return fn


def _elsewhere(device) -> bool:
    """Another device is the current one."""
    return device.index != torch._C._cuda_getDevice()


def _stream(device) -> int:
    """The device's current stream, without the object around it (2.3 us of a call of 10)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def slab_rows(m: int, n: int, top: int) -> int:
    """Rows of ``m`` that ``score`` takes at a time, where there is room."""
    return min(m, SLAB_ROWS if not top else max(256, SLAB_ELEMS // n // 256 * 256))


def work_bytes(m: int, n: int, k: int, top: int, i8: bool, sms: int = 148) -> int:
    """Workspace of ``score`` (``score_i8``) for ``m`` rows of ``k`` against ``n`` columns, for the memory plan: ``b2_score_work`` of a slab, or
    a little more.  16 bytes for every part of a row (tiles of 256 columns, up to 512 rows ranges of them instead), the token's logit, with
    alternatives the logits and a maximum of every 32, int8 rows and their scales."""
    rows, chunks = slab_rows(m, n, top), (n + 31) // 32
    parts = max(min(rows, 512) * min(sms, chunks), rows * ((n + 255) // 256) if rows > 512 else 0)
    return 16 * parts + 4 * rows + (4 * 33 * chunks * rows if top else 0) + ((k + 15) // 16 * 16 + 4) * rows * i8 + 512


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: Optional[int] = None, out: Optional[Logprobs] = None) -> Logprobs:
    """Rows of fp32 ``logits`` ``[m][vocabulary]`` (any row stride), one int32 token each.  ``out``: results to write, whose width is
    then ``top``."""
    m, n, ld, at = _rows_of(logits, torch.float32, "logits")
    dev = logits.device
    if n < 1:
        raise ValueError("logits of an empty vocabulary")
    _check_tokens(tokens, m, dev)
    out = _results(m, top, out, dev)
    if not m:
        return out
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top, out)
    K._check(_entry("b2_logprob_rows", "pliipippppp")(
        at, ld, m, n, tokens.data_ptr(), out.top_ids.shape[1], out.logprob.data_ptr(), out.entropy.data_ptr(),
        out.top_ids.data_ptr(), out.top_logprobs.data_ptr(), _stream(dev)), "logprob_rows")
    return out


def _score(x, w, w_scale, tokens, top: Optional[int], out: Optional[Logprobs]) -> Logprobs:
    i8, dev = w_scale is not None, x.device
    m, k, ldx, px = _rows_of(x, torch.bfloat16, "rows", 16)
    n, kw, ldw, pw = _rows_of(w, torch.int8 if i8 else torch.bfloat16, "head", 16)
    if kw != k or n < 1 or w.device != dev:
        raise ValueError(f"head {tuple(w.shape)} on {w.device} against rows {tuple(x.shape)} on {dev}")
    if k * (1 if i8 else 2) < 128 or i8 and k > MAX_I8_COLUMNS:
        raise ValueError(f"rows of {k} columns: 128 bytes of the head's type at least" + (f", {MAX_I8_COLUMNS} at most" if i8 else ""))
    _check_tokens(tokens, m, dev)
    out = _results(m, top, out, dev)
    if not m:
        return out
    top = out.top_ids.shape[1]
    room, run = _entry("b2_score_work", "iiiii", ctypes.c_longlong), _entry("b2_score", "plplpiiipipppppp")
    step = slab_rows(m, n, top)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _score(x, w, w_scale, tokens, None, out)
    while True:
        need = room(step, n, k, top, i8)
        if m % step:
            need = max(need, room(m % step, n, k, top, i8))
        try:
            work = torch.empty(need, dtype=torch.float32, device=dev)
            break
        except torch.OutOfMemoryError:
            if step <= 256 or not top:
                raise
            step = max(256, step // 512 * 256)      # fewer logits at a time
    ps, pt, pwork, stream = w_scale.data_ptr() if i8 else None, tokens.data_ptr(), work.data_ptr(), _stream(dev)
    for i in range(0, m, step):
        c = min(step, m - i)
        o = out if c == m else out.rows(i, i + c)
        K._check(run(px + 2 * i * ldx, ldx, pw, ldw, ps, c, n, k, pt + 4 * i, top, pwork, o.logprob.data_ptr(), o.entropy.data_ptr(),
                     o.top_ids.data_ptr(), o.top_logprobs.data_ptr(), stream), "score")
        K.launch_count += 2 if i8 else 1      # rows quantised; a row's parts joined
    return out


def score(x: torch.Tensor, head: torch.Tensor, tokens: torch.Tensor, top: Optional[int] = None, out: Optional[Logprobs] = None) -> Logprobs:
    """Rows ``x`` ``[m][k]`` against the lm_head ``[vocabulary][k]``, both bf16 with rows at multiples of 16 bytes: ``token_logprobs`` of
    ``x @ head.T`` in fp32."""
    return _score(x, head, None, tokens, top, out)


def score_i8(x: torch.Tensor, head: tuple, tokens: torch.Tensor, top: Optional[int] = None, out: Optional[Logprobs] = None) -> Logprobs:
    """Rows ``x`` ``[m][k]`` bf16 against an int8 lm_head (``[vocabulary][k]``, fp32 scale per row), rows of both at multiples of 16
    bytes: rows are quantised per token (s = max|x| / 127, q = rint(x (1 / s)) with the inverse rounded to fp32, as the int8 prompt pass does)
    and logits are (q . w) s s_w."""
    w8, scale = head
    if scale.dtype is not torch.float32 or scale.shape != (w8.shape[0],) or scale.device != x.device or not scale.is_contiguous():
        raise ValueError(f"scales of the head: {w8.shape[0]} contiguous fp32 numbers on {x.device}")
    return _score(x, w8, scale, tokens, top, out)
