"""Operators on device tensors over the C-ABI (include/gpullama3_hip.h, csrc/gl3_ops.hip): rows in 8-bit integers with a scale each, their
products, and log probabilities of tokens.  They take torch tensors of the GPU, run on torch's current stream of the tensors' device and may be
captured into a graph.  Forward only.  Nothing here computes and there is no fallback: CPU tensors are refused.

    w = quantize_rows(weight)                       # once: int8 codes [out, in] and a scale per channel
    logits = int8_linear(hidden, w, dtype=torch.float32)
    lp = token_logprobs(logits, targets, top=5)     # lp.logprob, lp.rank, lp.entropy, lp.top_ids, lp.top_logprobs
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import hip

CODE_BLOCK = 128             # GL3_CODE_BLOCK
MAX_K = 131071               # GL3_INT8_MAX_K
MAX_TOP = 64                 # GL3_LOGPROBS_MAX_TOP


def _bad(what):
    return hip.Gl3Error(hip.E_ARG, what)


_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _forward_only(t, name):
    """No derivative is lost in silence, of either mode (no_grad stops gradients only)."""
    if t.requires_grad and torch.is_grad_enabled():
        raise _bad(name + " requires a gradient: these operators are forward only")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise _bad(name + " has a tangent: these operators are forward only")


class Int8Rows:
    """Rows of int8 codes with a scale each; row i stands for codes[i, :cols] * scale[i].  codes: int8 [rows, ld], ld >= cols rounded up to a
    multiple of CODE_BLOCK, rows that start on 16 bytes, zeros from column cols to that multiple; scale: float32 [rows].  Checked once, here."""
    __slots__ = ("codes", "scale", "cols", "rows", "ld", "device")

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, cols: int):
        if codes.dim() != 2 or codes.dtype != torch.int8 or (codes.stride(1) != 1 and codes.shape[1] != 1):
            raise _bad("codes must be an int8 matrix with contiguous rows")
        if not 0 < cols <= MAX_K or codes.shape[1] < -(-cols // CODE_BLOCK) * CODE_BLOCK:
            raise _bad("a row of codes is %d columns and zeros up to a multiple of %d, at most %d" % (cols, CODE_BLOCK, MAX_K))
        if scale.dim() != 1 or scale.shape[0] != codes.shape[0] or scale.dtype != torch.float32 or scale.device != codes.device or not scale.is_contiguous():
            raise _bad("scale must hold one float32 per row of codes, beside them")
        _forward_only(scale, "scale")
        self.codes, self.scale, self.cols = codes, scale, cols
        self.rows, self.device = codes.shape[0], codes.device
        self.ld = codes.stride(0) if self.rows > 1 else codes.shape[1] // 16 * 16

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        return (self.codes[:, :self.cols].float() * self.scale[:, None]).to(dtype)


class TokenLogprobs(NamedTuple):
    """Per row: logprob (float32) and rank (int32, 1 = most probable) of the given token (None without targets), entropy (float32, None if not
    wanted), and the `top` most probable tokens: ids (int32, -1 behind the last one) and log probabilities (None for top = 0)."""
    logprob: Optional[torch.Tensor]
    rank: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def _rows(x, name):
    """A float matrix on a GPU whose rows are contiguous -> its row stride."""
    if not x.is_cuda:
        raise _bad(name + " must be on a GPU: there is no CPU path")
    if x.dim() != 2 or x.dtype not in _TYPES:
        raise _bad(name + " must be a matrix of float32, float16 or bfloat16")
    rows, inner = x.stride()
    if inner != 1 and x.shape[1] != 1:
        raise _bad(name + ": the elements of a row must be contiguous")
    _forward_only(x, name)
    return rows


def _like(t, name, shape, dtype, device):
    if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise _bad("%s must be a contiguous %s tensor of shape %s on %s" % (name, dtype, tuple(shape), device))


@functools.lru_cache(maxsize=4096)
def _int8_bytes(m, n, k):
    a, b = C.c_uint64(), C.c_uint64()
    hip.check(hip.lib().gl3_int8_workspace(m, n, k, C.byref(a), C.byref(b)))
    return a.value, b.value


@functools.lru_cache(maxsize=4096)
def _logprobs_bytes(rows, vocab, top):
    a = C.c_uint64()
    hip.check(hip.lib().gl3_logprobs_workspace(rows, vocab, top, C.byref(a)))
    return a.value


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _call(fn, device, *args):
    code = fn(device.index, torch._C._cuda_getCurrentRawStream(device.index), *args)
    if code:
        hip.check(code)


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """float rows [rows, cols] -> Int8Rows: scale = max |x| / 127, code = rint(x * (127 / max |x|)) in float32.  A row of zeros (or below 2^-100) has
    scale 0; a row with a NaN or an infinity has scale NaN."""
    ld = _rows(x, "x")
    rows, cols = x.shape
    if not 0 < cols <= MAX_K:
        raise _bad("x must have 1 .. %d columns" % MAX_K)
    device = x.device
    ld_codes = -(-cols // CODE_BLOCK) * CODE_BLOCK
    codes = torch.empty(rows, ld_codes, dtype=torch.int8, device=device)
    scale = torch.empty(rows, dtype=torch.float32, device=device)
    _call(hip.lib().gl3_quantize_rows, device, x.data_ptr(), _TYPES[x.dtype], rows, cols, ld, codes.data_ptr(), ld_codes, scale.data_ptr())
    r = Int8Rows.__new__(Int8Rows)          # (made here: nothing to check)
    r.codes, r.scale, r.cols, r.rows, r.ld, r.device = codes, scale, cols, rows, ld_codes, device
    return r


def _result(w, bias, m, k, dtype, out, device):
    n = w.rows
    if w.cols != k or w.device != device:
        raise _bad("the rows have %d columns on %s, the weights %d on %s" % (k, device, w.cols, w.device))
    if dtype not in _TYPES:
        raise _bad("results are float32, float16 or bfloat16")
    _forward_only(w.scale, "scale")
    if bias is not None:
        _like(bias, "bias", (n,), torch.float32, device)
        _forward_only(bias, "bias")
    if out is None:
        return torch.empty(m, n, dtype=dtype, device=device), n
    _forward_only(out, "out")
    if out.shape != (m, n) or out.dtype != dtype or out.device != device or (out.stride(1) != 1 and n != 1):
        raise _bad("out must be a %d x %d matrix of %s with contiguous rows on %s" % (m, n, dtype, device))
    return out, out.stride(0)


def _meet(p, p_rows, p_pitch, p_width, q, q_rows, q_pitch, q_width):
    """Whether two matrices, each given by address, rows, bytes between rows and bytes of a row, share a byte (of different pitches: may share one)."""
    if p + (p_rows - 1) * p_pitch + p_width <= q or q + (q_rows - 1) * q_pitch + q_width <= p:
        return False
    pitch = q_pitch if p_rows == 1 else p_pitch
    if p_rows == q_rows == 1 or (q_rows > 1 and q_pitch != pitch):
        return True
    gap = (q - p) % pitch          # columns of one buffer, side by side
    return not (p_width <= gap and gap + q_width <= pitch)


def _apart(out, m, n, ldy, x, ldx, k, bias):
    """Workgroups write results while others still read: out must not lie over an input."""
    size = out.element_size()
    y = (out.data_ptr(), m, ldy * size, n * size)
    if x is not None and _meet(*y, x.data_ptr(), m, ldx * x.element_size(), k * x.element_size()):
        raise _bad("out overlaps x")
    if bias is not None and _meet(*y, bias.data_ptr(), 1, 0, 4 * n):
        raise _bad("out overlaps bias")


def _written(out):
    """out= has been written in place: a backward pass that has saved it finds that."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out


def int8_matmul(a: Int8Rows, w: Int8Rows, bias: Optional[torch.Tensor] = None, dtype=torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[i, j] = (sum_k a[i, k] w[j, k]) * a.scale[i] * w.scale[j] (+ bias[j]): the sum exact in int32, one rounding to dtype.
    out: a matrix of dtype with contiguous rows that the results are written to (apart from the inputs)."""
    device = a.device
    if device.type != "cuda":
        raise _bad("a must be on a GPU: there is no CPU path")
    m, k, n = a.rows, a.cols, w.rows
    _forward_only(a.scale, "scale")
    y, ldy = _result(w, bias, m, k, dtype, out, device)
    if out is not None and bias is not None and m and n:
        _apart(y, m, n, ldy, None, 0, 0, bias)
    nbytes = _int8_bytes(m, n, k)[0]
    ws = _workspace(nbytes, device)
    _call(hip.lib().gl3_int8_matmul, device, a.codes.data_ptr(), a.ld, a.scale.data_ptr(), w.codes.data_ptr(), w.ld, w.scale.data_ptr(), _ptr(bias), m, n, k,
          y.data_ptr(), _TYPES[dtype], ldy, _ptr(ws), nbytes)
    return y if out is None else _written(out)


def int8_linear(x: torch.Tensor, w: Int8Rows, bias: Optional[torch.Tensor] = None, dtype=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int8_matmul(quantize_rows(x), w, bias), bit for bit, in as few launches as the sizes allow (one up to 4 tokens, 8 where k <= 2048, of matrices that are
    not too wide: several products of such rows want a linear each, of more rows one quantize_rows).  dtype: of the result (default: x's).
    out: as in int8_matmul."""
    ldx = _rows(x, "x")
    m, k = x.shape
    n = w.rows
    device = x.device
    if dtype is None:
        dtype = x.dtype
    y, ldy = _result(w, bias, m, k, dtype, out, device)
    if out is not None and m and n:
        _apart(y, m, n, ldy, x, ldx, k, bias)
    nbytes = _int8_bytes(m, n, k)[1]
    ws = _workspace(nbytes, device)
    _call(hip.lib().gl3_int8_linear, device, x.data_ptr(), _TYPES[x.dtype], ldx, w.codes.data_ptr(), w.ld, w.scale.data_ptr(), _ptr(bias), m, n, k,
          y.data_ptr(), _TYPES[dtype], ldy, _ptr(ws), nbytes)
    return y if out is None else _written(out)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0, entropy: bool = True) -> TokenLogprobs:
    """Log probability and rank of targets[r] (int32; negative: no token is given, 0 and rank 0) under softmax(logits[r]), the row's entropy, and its
    `top` most probable tokens, lower id first among equal logits.  See gl3_token_logprobs for rows with infinities or NaN."""
    ld = _rows(logits, "logits")
    rows, vocab = logits.shape
    device = logits.device
    if vocab < 1 or not 0 <= top <= MAX_TOP:
        raise _bad("vocab must be positive, top in 0 .. %d" % MAX_TOP)
    logprob = rank = ent = ids = values = None
    if targets is not None:
        _like(targets, "targets", (rows,), torch.int32, device)
        logprob, rank = torch.empty(rows, dtype=torch.float32, device=device), torch.empty(rows, dtype=torch.int32, device=device)
    if entropy:
        ent = torch.empty(rows, dtype=torch.float32, device=device)
    if top:
        ids, values = torch.empty(rows, top, dtype=torch.int32, device=device), torch.empty(rows, top, dtype=torch.float32, device=device)
    nbytes = _logprobs_bytes(rows, vocab, top)
    ws = _workspace(nbytes, device)
    _call(hip.lib().gl3_token_logprobs, device, logits.data_ptr(), _TYPES[logits.dtype], rows, vocab, ld, _ptr(targets), top, _ptr(logprob), _ptr(rank), _ptr(ent), _ptr(ids),
          _ptr(values), _ptr(ws), nbytes)
    return TokenLogprobs(logprob, rank, ent, ids, values)
