"""The gated delta rule layer's core for many sequences at once (csrc/lxm_seq.hip, C ABI include/lxm_seq.h):
a batch of prompts, of single tokens, or of both, each sequence's recurrent states and convolution window in a
slot of caches that all share.

    s = Sequences([2048, 1, 7], slots=[4, 0, 2])           # lengths, on the host; kept while they hold
    y = short_conv(x, w, window, s)                        # (N, C): 4 taps, SiLU; window advanced
    o = gated_delta(q, k, v, g, beta, state, s)            # (N, nv, V); state advanced

The tokens of the batch lie one sequence after another. Both functions run on the tensors' device and the
current stream, can be captured in a graph (the sequences' tables are the plan's), and give no gradients.
Where chunk.gated_delta_chunked runs one sequence of the stack's own padded shape, this takes the layer's
tensors as they are: bf16, fp16 or fp32, un-normalised, strided views of a projection's output.
"""

from __future__ import annotations

import ctypes
from array import array

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import mk_build

CHUNK = 64              # positions per chunk (LXM_SEQ_CHUNK)
# The longest sequences that go through the recurrence position by position: in calls of fewer than MANY_HEADS
# (sequence, value head) pairs, and of more in bf16 and in fp16 and fp32 (whose chunks are split into more
# products). 128 x 128, 32 heads, equal lengths, recurrence against chunks in us, of 1, 8 and 60 sequences:
# 8 positions bf16 16 and 18, 20 and 33, 66 and 143; 12 bf16 22 and 18, fp32 21 and 21; 16 bf16 28 and 18, 32
# and 32, 106 and 146; 24 bf16 40 and 18, 45 and 33, 148 and 155, fp16 41 and 19, 45 and 45, 149 and 253,
# fp32 39 and 21, 45 and 49, 140 and 341; 32 fp32 50 and 21, 60 and 49, 181 and 345.
RECURRENT_MAX, MANY_HEADS = 8, 256
RECURRENT_MAX_MANY = {torch.bfloat16: 16, torch.float16: 24, torch.float32: 24}
WS_MAX = 192 << 20      # a call's workspace, unless one chunk needs more; more chunks go in groups
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}

_P, _L, _I = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32


class SeqTable(ctypes.Structure):
    _fields_ = [(n, _P) for n in ("seqs", "chunks")] + \
        [(n, _I) for n in ("n_seqs", "n_tokens", "n_chunks", "max_len")]


class ConvIO(ctypes.Structure):
    _fields_ = [(n, _P) for n in ("x", "w", "window", "y")] + \
        [(n, _L) for n in ("x_ts", "w_ss", "y_ts")] + [(n, _I) for n in ("C", "type")]


class GdIO(ctypes.Structure):
    _fields_ = [(n, _P) for n in ("q", "k", "v", "g", "beta", "state", "o")] + \
        [(n, _L) for n in ("q_ts", "q_hs", "k_ts", "k_hs", "v_ts", "v_hs", "g_ts", "g_hs", "b_ts",
                           "b_hs", "s_ss", "o_ts", "o_hs")] + \
        [(n, _I) for n in ("nk", "r", "K", "V", "type", "beta_type", "unit")] + [("scale", ctypes.c_float)]


class Sequences:
    """The sequences of a batch: their lengths (>= 0) and the slots of the caches they read and leave their
    state in. Slots of one batch are distinct; slot -1 (any number of them) starts from zeros and keeps
    nothing: padding, or a sequence that ends with the call. Default: slots 0, 1, 2, ... Lengths and slots are
    host integers, checked here; the tables go to the device once, by a copy that waits. A graph that captured
    a call reads the tables at every replay: the plan is to live as long."""

    def __init__(self, lengths, slots=None, device="cuda"):
        lens = [int(n) for n in lengths]
        slots = list(range(len(lens))) if slots is None else [int(s) for s in slots]
        if len(slots) != len(lens):
            raise ValueError(f"{len(lens)} sequences and {len(slots)} slots")
        if lens and min(lens) < 0:
            raise ValueError("a sequence of negative length")
        used = [s for s in slots if s >= 0]
        if len(set(used)) != len(used) or (slots and min(slots) < -1):
            raise ValueError("slots: distinct, or -1 for none")
        self.lengths, self.slots = tuple(lens), tuple(slots)
        self.n_seqs, self.n_tokens = len(lens), sum(lens)
        self.max_len, self.max_slot = max(lens, default=0), max(slots, default=-1)
        if self.n_tokens >= 1 << 31 or self.max_slot >= 1 << 31:
            raise ValueError("a batch holds less than 2^31 tokens and slots")
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device, self.index = dev, dev.index if dev.type == "cuda" else -1
        order = sorted(range(len(lens)), key=lens.__getitem__, reverse=True)  # (longest first)
        record = [0] * len(lens)
        for i, b in enumerate(order):
            record[b] = i
        seqs, chunks, first = [None] * len(lens), array("i"), 0
        for b, n in enumerate(lens):
            seqs[record[b]] = (slots[b], first, first + n, len(chunks) // 4)
            for t in range(0, n, CHUNK):
                chunks.extend((first + t, min(CHUNK, n - t), record[b], t // CHUNK))
            first += n
        self.n_chunks = len(chunks) // 4
        table = array("i")
        for q in seqs:
            table.extend(q)
        table.extend(chunks)
        # (a synchronous copy: the tables are there for whatever stream uses them)
        self.tables = (torch.frombuffer(table, dtype=torch.int32).view(-1, 4) if table else
                       torch.empty(0, 4, dtype=torch.int32)).to(dev, copy=True)
        self.stream = torch.cuda.current_stream(dev).cuda_stream if self.index >= 0 else None
        ptr = self.tables.data_ptr()
        self.table = SeqTable(ptr, ptr + 16 * len(lens), self.n_seqs, self.n_tokens, self.n_chunks,
                              self.max_len)

    def __repr__(self):
        return f"Sequences({self.n_seqs} of {self.n_tokens} tokens on {self.device})"


def _step(t, d):
    return t.stride(d) if t.shape[d] > 1 else 0


def _dense(t, d):
    """Whether dimensions d .. of t lie one element after another."""
    n = 1
    for i in range(t.dim() - 1, d - 1, -1):
        if t.shape[i] > 1 and t.stride(i) != n:
            return False
        n *= t.shape[i]
    return True


def _aligned(t):
    """Whether the rows of t (its last dimension) are dense and 16 bytes or a multiple apart."""
    a = 16 // t.element_size()
    return _dense(t, t.dim() - 1) and not any(_step(t, d) % a for d in range(t.dim() - 1))


def _vectors(t):
    return t if _aligned(t) and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _launch(seqs, f, *args):
    i = seqs.index
    if i < 0:
        raise ValueError(f"the batch kernels run on a GPU, not on {seqs.device}")
    stream = torch._C._cuda_getCurrentRawStream(i)
    if stream != seqs.stream:  # (the tables' memory is not given to others before this stream is through)
        seqs.tables.record_stream(torch.cuda.current_stream(i))
    if torch.cuda.current_device() == i:
        e = f(*args, stream)
    else:
        with torch.cuda.device(i):
            e = f(*args, stream)
    if e:
        raise RuntimeError(f"{f.__name__} failed: hipError {e}")


def refuse_gradients(*tensors):
    """What needs a gradient, backward or forward, while gradients are formed at all, is refused (None is skipped)."""
    for t in tensors:
        if t is not None and (torch.is_grad_enabled() and t.requires_grad or
                              forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError("no gradients are formed here: call under torch.no_grad(), without tangents")


def _refuse(seqs, *tensors):
    """Tensors elsewhere than the sequences or with gradients to be formed (None is skipped)."""
    for t in tensors:
        if t is not None and t.device != seqs.device:
            raise ValueError(f"a tensor on {t.device}, the sequences on {seqs.device}")
    refuse_gradients(*tensors)


def _written(*tensors):
    """Tells autograd that the kernels change these in place: what saved one for its backward pass fails there instead
    of taking the new values."""
    for t in tensors:
        if not t.is_inference():
            increment_version(t)


_calls = {}  # what calls of given shapes, strides and types pass on, their checks done


def _remember(key, value):
    if len(_calls) >= 256:
        _calls.clear()
    _calls[key] = value
    return value


def _fits(seqs, rows, slots):
    if seqs.n_tokens > rows:
        raise ValueError(f"{rows} rows for {seqs.n_tokens} tokens")
    if seqs.max_slot >= slots:
        raise ValueError(f"slot {seqs.max_slot} of a cache of {slots}")


def _check_out(out, like, what):
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"out: {what} as the input's, {tuple(like.shape)} {like.dtype}")


def _apart(out):
    """Refuses a tensor two of whose elements may share memory: a dimension's step is past all that lies within it."""
    end = 0
    for step, n in sorted((out.stride(d), out.shape[d]) for d in range(out.dim()) if out.shape[d] > 1):
        if step <= end:
            raise ValueError("out: elements that share memory")
        end += (n - 1) * step


def _new_out(like, seqs):
    out = like.new_empty(like.shape)
    if like.dim() and like.shape[0] > seqs.n_tokens:
        out[seqs.n_tokens:].zero_()
    return out


def short_conv(x, w, window, seqs, out=None):
    """The causal convolution before the delta rule: y_t = silu(sum_j w[:, j] x_{t - 3 + j}) for every
    sequence of the batch, the inputs before its first from its window, which afterwards holds its last four
    inputs. x (N, C), N >= the sequences' tokens, any row stride; w (C, 4); window (slots, C, 4), updated in
    place (the stack's own conv states: conv_states[0] with the batch as slots); all of one type (bf16, fp16
    or fp32). Sums in float32, rounded once. Returns (N, C), rows past the last sequence zero; with out (which
    must not overlap x) those rows are left as they were."""
    i = seqs.index
    if x.get_device() != i or w.get_device() != i or window.get_device() != i or \
            (out is not None and (out.get_device() != i or out.requires_grad)) or \
            forward_ad._current_level >= 0 or \
            (torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or window.requires_grad)):
        _refuse(seqs, x, w, window, out)
    if out is not None:
        _check_out(out, x, "x")
    y = _new_out(x, seqs) if out is None else out
    key = (x.shape, x.stride(), x.dtype, w.shape, w.stride(), w.dtype, window.shape, window.stride(),
           window.dtype, y.stride())
    io = _calls.get(key)
    if io is None:
        io = _remember(key, _conv_io(x, w, window, y))
    _fits(seqs, x.shape[0], window.shape[0])
    if seqs.n_tokens == 0:
        return y
    if io is False:  # (columns that do not lie side by side)
        z = short_conv(x.contiguous(), w.contiguous(), window, seqs)
        y[:seqs.n_tokens] = z[:seqs.n_tokens]
        return y
    io = ConvIO.from_buffer_copy(io)
    io.x, io.w, io.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
    io.window = window.data_ptr() or io.y  # (a cache of no slots has no address, and none is read)
    _launch(seqs, mk_build.load().lxm_short_conv, ctypes.byref(seqs.table), ctypes.byref(io))
    _written(*((window,) if out is None else (window, out)))
    return y


def _conv_io(x, w, window, y):
    if x.dim() != 2 or x.dtype not in TYPES or w.dtype != x.dtype or window.dtype != x.dtype:
        raise ValueError("short_conv: x (N, C), w and window of one type: bf16, fp16 or fp32")
    C = x.shape[1]
    if w.shape != (C, 4) or window.dim() != 3 or window.shape[1:] != (C, 4) or C < 1:
        raise ValueError("short_conv: x (N, C), w (C, 4), window (slots, C, 4)")
    if not _dense(window, 1) or (window.shape[0] > 1 and window.stride(0) < 4 * C):
        raise ValueError("short_conv: a slot's window is dense, and the slots lie apart")
    _apart(y)
    if not (_dense(x, 1) and _dense(w, 0) and _dense(y, 1)):
        return False
    return ConvIO(0, 0, 0, 0, _step(x, 0), _step(window, 0), _step(y, 0), C, TYPES[x.dtype])


def gated_delta(q, k, v, g, beta, state, seqs, scale=None, unit=True, out=None):
    """The gated delta rule over every sequence of the batch, position by position
        S <- exp(g) S;  d = beta (v - S^T k);  S <- S + k d^T;  o = scale S^T q
    with S the sequence's state (state[slot, head], updated in place). q, k (N, nk, K), v (N, nv, V) of one
    type (bf16, fp16 or fp32), K 64, 128 or 256, V a multiple of 16 up to 256, nv a multiple of nk (value head
    h reads key head h // (nv // nk)); g (N, nv) float32 log decays (-inf forgets), beta (N, nv) float32 or v's
    type; state (slots, nv, K, V) float32, a slot dense. N >= the sequences' tokens. unit: q and k are divided
    by sqrt(sum of squares + 1e-6) first; scale: K ** -0.5 unless given. Returns o (N, nv, V), v's type; rows
    past the last sequence as in short_conv; out must not overlap the inputs.

    Products and sums are float32's (in chunks, of numbers below 2^-110 only the leading digits count). Batches
    whose longest sequence has more than 8 positions (in large batches 16 in bfloat16, 24 in the others) go in
    chunks of 64 on the matrix cores, with a workspace of up to WS_MAX bytes for the call (or what two states of
    all heads and one chunk take: lxm_gd_ws); there, as in every chunked form, a NaN or infinity reaches the
    other positions of its chunk. A view whose rows are not 16-byte aligned is copied first."""
    i = seqs.index
    if q.get_device() != i or k.get_device() != i or v.get_device() != i or g.get_device() != i or \
            beta.get_device() != i or state.get_device() != i or \
            (out is not None and (out.get_device() != i or out.requires_grad)) or \
            forward_ad._current_level >= 0 or (torch.is_grad_enabled() and (
                q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or
                beta.requires_grad or state.requires_grad)):
        _refuse(seqs, q, k, v, g, beta, state, out)
    if out is not None:
        _check_out(out, v, "v")
    o = _new_out(v, seqs) if out is None else out
    scale, unit = None if scale is None else float(scale), bool(unit)  # (values: a tensor's may change)
    key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype,
           g.shape, g.stride(), g.dtype, beta.shape, beta.stride(), beta.dtype, state.shape,
           state.stride(), state.dtype, o.stride(), scale, unit)
    io = _calls.get(key)
    if io is None:
        io = _remember(key, _delta_io(q, k, v, g, beta, state, o, scale, unit))
    _fits(seqs, q.shape[0], state.shape[0])
    if seqs.n_tokens == 0:
        return o
    p = (q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(),
         o.data_ptr())
    if p[5] % 16:
        raise ValueError("gated_delta: a slot's state is 16-byte aligned")
    if io is False or (p[0] | p[1] | p[2] | p[6]) % 16:  # (rows that do not start at 16 bytes)
        z = gated_delta(_vectors(q), _vectors(k), _vectors(v), g, beta, state, seqs, scale, unit)
        o[:seqs.n_tokens] = z[:seqs.n_tokens]
        return o
    io = GdIO.from_buffer_copy(io)
    io.q, io.k, io.v, io.g, io.beta, io.state, io.o = p
    io.state = p[5] or p[6]  # (a cache of no slots has no address, and none is read)
    lib = mk_build.load()
    if seqs.max_len <= (RECURRENT_MAX if seqs.n_seqs * v.shape[1] < MANY_HEADS else
                        RECURRENT_MAX_MANY[v.dtype]):
        _launch(seqs, lib.lxm_gd_recurrent, ctypes.byref(seqs.table), ctypes.byref(io))
    else:
        n, least = _L(), _L()
        lib.lxm_gd_ws(ctypes.byref(io), seqs.n_chunks, ctypes.byref(n))
        lib.lxm_gd_ws(ctypes.byref(io), 1, ctypes.byref(least))
        n = max(least.value, min(n.value, WS_MAX))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        _launch(seqs, lib.lxm_gd_chunks, ctypes.byref(seqs.table), ctypes.byref(io), ws.data_ptr(), n)
    _written(*((state,) if out is None else (state, out)))
    return o


def _delta_io(q, k, v, g, beta, state, o, scale, unit):
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[0] != q.shape[0]:
        raise ValueError("gated_delta: q, k (N, nk, K), v (N, nv, V)")
    N, nk, K = q.shape
    nv, V = v.shape[1:]
    if q.dtype not in TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("gated_delta: q, k and v of one type: bf16, fp16 or fp32")
    if K not in (64, 128, 256) or V < 16 or V > 256 or V % 16:
        raise ValueError(f"gated_delta: {K} key dims (64, 128 or 256), {V} value dims (a multiple of 16, "
                         "up to 256)")
    if nk < 1 or nv < 1 or nv % nk:
        raise ValueError(f"gated_delta: {nv} value heads on {nk} key heads")
    if g.shape != (N, nv) or g.dtype != torch.float32 or beta.shape != (N, nv) or \
            beta.dtype not in (torch.float32, v.dtype):
        raise ValueError("gated_delta: g (N, nv) float32, beta (N, nv) float32 or v's type")
    if state.dim() != 4 or state.shape[1:] != (nv, K, V) or state.dtype != torch.float32:
        raise ValueError("gated_delta: state (slots, nv, K, V) float32")
    if not _dense(state, 1) or _step(state, 0) % 4 or \
            (state.shape[0] > 1 and state.stride(0) < nv * K * V):
        raise ValueError("gated_delta: a slot's state is dense and 16-byte aligned, and the slots lie apart")
    _apart(o)
    if not (_aligned(q) and _aligned(k) and _aligned(v) and _aligned(o)):
        return False
    return GdIO(0, 0, 0, 0, 0, 0, 0, _step(q, 0), _step(q, 1), _step(k, 0), _step(k, 1), _step(v, 0),
                _step(v, 1), g.stride(0), g.stride(1), beta.stride(0), beta.stride(1), _step(state, 0),
                _step(o, 0), _step(o, 1), nk, nv // nk, K, V, TYPES[v.dtype], TYPES[beta.dtype],
                int(unit), K ** -0.5 if scale is None else scale)
