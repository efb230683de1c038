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

from . import hip

CODE_BLOCK = 128             # GL3_CODE_BLOCK
MAX_K = 131071               # GL3_INT8_MAX_K
MAX_TOP = 64                 # GL3_LOGPROBS_MAX_TOP
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class Int8Rows(NamedTuple):
    """Rows of int8 codes with a scale each; row i stands for codes[i, :cols] * scale[i].  codes: int8 [rows, ld], ld >= cols rounded up to a
    multiple of CODE_BLOCK and a multiple of 16, zeros from column cols to that multiple; scale: float32 [rows]."""
    codes: torch.Tensor
    scale: torch.Tensor
    cols: int

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


def _need(ok, what):
    if not ok:
        raise hip.Gl3Error(hip.E_ARG, what)


def _rows(x, name):
    """A float matrix on a GPU whose rows are contiguous -> its row stride."""
    _need(x.is_cuda, name + " must be on a GPU: there is no CPU path")
    _need(x.dim() == 2 and x.dtype in _TYPES, name + " must be a matrix of float32, float16 or bfloat16")
    _need(x.stride(1) == 1 or x.shape[1] == 1, name + ": the elements of a row must be contiguous")
    _need(not (x.requires_grad and torch.is_grad_enabled()), name + " requires a gradient: these operators are forward only")
    return x.stride(0)


def _like(t, name, shape, dtype, device):
    _need(t.shape == shape and t.dtype == dtype and t.device == device and t.is_contiguous(), "%s must be a contiguous %s tensor of shape %s on %s" % (name, dtype, tuple(shape), device))


def _codes(r, name, device):
    c = r.codes
    _need(c.dim() == 2 and c.dtype == torch.int8 and c.device == device and c.stride(1) == 1, name + ".codes must be an int8 matrix with contiguous rows on " + str(device))
    _need(0 < r.cols <= MAX_K and c.shape[1] >= -(-r.cols // CODE_BLOCK) * CODE_BLOCK, name + ".codes: a row is cols columns and zeros up to a multiple of %d" % CODE_BLOCK)
    s = r.scale
    _need(s.dim() == 1 and s.shape[0] == c.shape[0] and s.dtype == torch.float32 and s.device == device and s.is_contiguous(), name + ".scale must hold one float32 per row on " + str(device))
    return c.stride(0) if c.shape[0] > 1 else c.shape[1]


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
    _need(0 < cols <= MAX_K, "x must have 1 .. %d columns" % MAX_K)
    codes = torch.empty(rows, -(-cols // CODE_BLOCK) * CODE_BLOCK, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call(hip.lib().gl3_quantize_rows, x.device, x.data_ptr(), _TYPES[x.dtype], rows, cols, ld, codes.data_ptr(), codes.shape[1], scale.data_ptr())
    return Int8Rows(codes, scale, cols)


def _product(w, bias, m, k, dtype, out, device):
    ldw = _codes(w, "w", device)
    n = w.codes.shape[0]
    _need(w.cols == k, "the rows have %d columns, the weights %d" % (k, w.cols))
    _need(dtype in _TYPES, "results are float32, float16 or bfloat16")
    if bias is not None:
        _like(bias, "bias", (n,), torch.float32, device)
    if out is None:
        out = torch.empty(m, n, dtype=dtype, device=device)
    else:
        _need(out.shape == (m, n) and out.dtype == dtype and out.device == device and (out.stride(1) == 1 or n == 1), "out must be a %d x %d matrix of %s with contiguous rows on %s" % (m, n, dtype, device))
    return ldw, n, out


def int8_matmul(a: Int8Rows, w: Int8Rows, bias: Optional[torch.Tensor] = None, dtype=torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[i, j] = (sum_k a[i, k] w[j, k]) * a.scale[i] * w.scale[j] (+ bias[j]): the sum exact in int32, one rounding to dtype."""
    device = a.codes.device
    _need(device.type == "cuda", "a must be on a GPU: there is no CPU path")
    lda = _codes(a, "a", device)
    m, k = a.codes.shape[0], a.cols
    ldw, n, out = _product(w, bias, m, k, dtype, out, device)
    nbytes = _int8_bytes(m, n, k)[0]
    ws = _workspace(nbytes, device)
    _call(hip.lib().gl3_int8_matmul, device, a.codes.data_ptr(), lda, a.scale.data_ptr(), w.codes.data_ptr(), ldw, w.scale.data_ptr(), _ptr(bias), m, n, k,
          out.data_ptr(), _TYPES[dtype], out.stride(0), _ptr(ws), nbytes)
    return out


def int8_linear(x: torch.Tensor, w: Int8Rows, bias: Optional[torch.Tensor] = None, dtype=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int8_matmul(quantize_rows(x), w, bias), bit for bit, in as few launches as the sizes allow.  dtype: of the result (default: x's)."""
    ldx = _rows(x, "x")
    m, k = x.shape
    device = x.device
    dtype = x.dtype if dtype is None else dtype
    ldw, n, out = _product(w, bias, m, k, dtype, out, device)
    nbytes = _int8_bytes(m, n, k)[1]
    ws = _workspace(nbytes, device)
    _call(hip.lib().gl3_int8_linear, device, x.data_ptr(), _TYPES[x.dtype], ldx, w.codes.data_ptr(), ldw, w.scale.data_ptr(), _ptr(bias), m, n, k,
          out.data_ptr(), _TYPES[dtype], out.stride(0), _ptr(ws), nbytes)
    return out


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0, entropy: bool = True) -> TokenLogprobs:
    """Log probability and rank of targets[r] (int32; negative: no token is given, 0 and rank 0) under softmax(logits[r]), the row's entropy, and its
    `top` most probable tokens, lower id first among equal logits.  See gl3_token_logprobs for rows with infinities or NaN."""
    ld = _rows(logits, "logits")
    rows, vocab = logits.shape
    device = logits.device
    _need(vocab > 0 and 0 <= top <= MAX_TOP, "vocab must be positive, top in 0 .. %d" % MAX_TOP)
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
