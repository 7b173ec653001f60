"""How sure a model is of given tokens (csrc/lxm_score.hip, C ABI include/lxm_score.h): beside the argmax of
Fast.head_argmax and of the decodes, the log probabilities of a text's own tokens, each row's entropy, the
token's rank and the best alternatives, in one pass over logits that a caller has.

    r = token_logprobs(logits, tokens, top=8)
    r.logprob, r.entropy, r.rank, r.top_tokens, r.top_logprobs
"""

from __future__ import annotations

import ctypes
import operator
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import mk_build
from .seqs import refuse_gradients

TOP_MAX = 64  # alternatives at most (LXM_SCORE_TOP)
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class ScoreIO(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("logits", "tokens", "logprob", "entropy", "rank",
                                               "top_tokens", "top_logprobs")] + \
        [("stride", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("rows", "V", "top", "type", "wide")]


class Scores(NamedTuple):
    logprob: torch.Tensor       # (N,) float32
    entropy: torch.Tensor       # (N,) float32, in nats
    rank: torch.Tensor          # (N,) int32
    top_tokens: torch.Tensor    # (N, min(top, V)) int32
    top_logprobs: torch.Tensor  # (N, min(top, V)) float32


def token_logprobs(logits, tokens, top=0):
    """The log probability of tokens[i] under the softmax of row i of logits (N, V) (bf16, fp16 or fp32; any
    row stride and alignment), the row's entropy, and the token's rank: how many tokens come before it by
    larger logit, then by lower token (0: the first maximum, the token that a greedy decode takes). top: that many
    of the first tokens in that order, with their log probabilities. tokens (N,) int32 or int64 on the same
    device; a negative one is none (padding): log probability 0, rank -1. One past V - 1: NaN and -1.

    Sums are float32's. A logit of -inf has probability 0. In a row of nothing but -inf, or with a NaN or +inf,
    the log probabilities and the entropy are NaN (as log_softmax has them); a NaN comes before every other
    logit in the order, and its own rank is -1. Runs on the current stream; no gradients."""
    i = logits.get_device()
    if tokens.get_device() != i:
        raise ValueError(f"token_logprobs: logits on {logits.device}, tokens on {tokens.device}")
    if logits.requires_grad or forward_ad._current_level >= 0:
        refuse_gradients(logits)
    top = operator.index(top)  # (its value: a tensor's may change)
    key = (logits.shape, logits.stride(), logits.dtype, tokens.shape, tokens.stride(), tokens.dtype, top, i)
    call = _calls.get(key)
    if call is None:
        call = _io(logits, tokens, top)
        if len(_calls) >= 64:
            _calls.clear()
        _calls[key] = call
    if call is False:  # (columns that do not lie side by side)
        return token_logprobs(logits.contiguous(), tokens.contiguous(), top)
    io, need = call
    N, k = io.rows, io.top
    # (tensors of their own: a caller may change one in place, keep or save it without the others)
    f32, i32 = torch.float32, torch.int32
    out = Scores(logits.new_empty(N, dtype=f32), logits.new_empty(N, dtype=f32), logits.new_empty(N, dtype=i32),
                 logits.new_empty((N, k), dtype=i32), logits.new_empty((N, k), dtype=f32))
    if N == 0:
        return out
    ws = logits.new_empty(need, dtype=torch.uint8) if need else None
    io = ScoreIO.from_buffer_copy(io)
    io.logits, io.tokens = logits.data_ptr(), tokens.data_ptr()
    io.logprob, io.entropy, io.rank, io.top_tokens, io.top_logprobs = [t.data_ptr() for t in out]
    args = (ctypes.byref(io), ws.data_ptr() if need else 0, need)
    f = mk_build.load().lxm_score
    if torch.cuda.current_device() == i:
        e = f(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            e = f(*args, torch._C._cuda_getCurrentRawStream(i))
    if e:
        raise RuntimeError(f"lxm_score failed: hipError {e}")
    return out


_calls = {}  # what a call of these shapes, strides and types passes on, its checks done


def _io(logits, tokens, top):
    if logits.dim() != 2 or logits.dtype not in TYPES or logits.shape[1] < 1:
        raise ValueError("token_logprobs: logits (N, V), bf16, fp16 or fp32")
    N, V = logits.shape
    if tokens.shape != (N,) or tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("token_logprobs: tokens (N,), int32 or int64")
    if top < 0 or top > TOP_MAX:
        raise ValueError(f"token_logprobs: {top} alternatives (0 to {TOP_MAX})")
    if V >= (1 << 31) - 64 or N >= 1 << 31:
        raise ValueError("token_logprobs: too many logits")
    if not logits.is_cuda:
        raise ValueError(f"token_logprobs runs on a GPU, not on {logits.device}")
    if (logits.stride(1) != 1 and V > 1) or (tokens.stride(0) != 1 and N > 1):
        return False
    io = ScoreIO(stride=logits.stride(0) if N > 1 else 0, rows=N, V=V, top=min(int(top), V),
                 type=TYPES[logits.dtype], wide=int(tokens.dtype == torch.int64))
    need = ctypes.c_int64()
    if mk_build.load().lxm_score_ws(ctypes.byref(io), ctypes.byref(need)):
        raise RuntimeError("lxm_score_ws failed")
    return io, need.value
