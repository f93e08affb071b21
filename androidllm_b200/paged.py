"""Operators of a batched step on device data: norms, rotation and the cache
write of new rows (``rope_append``), attention of ragged batches over a paged
cache (``attn_paged``), acceptance of drafted tokens (``verify``).

Tensors are device arrays of the caller: objects with ``data_ptr()``,
``shape``, ``stride()`` and ``dtype`` (torch tensors), objects with
``__cuda_array_interface__``, or ``DeviceArray`` views of memory of the
library.  Nothing here waits for the GPU: the calls run on the context's
stream (``ops.default_context(device, stream)`` gives a context on the
caller's own stream), can be captured into a CUDA graph, and a captured call
reads the lengths, page numbers and draws that its device arrays hold when it
is replayed.  What the device finds out of range is reported by the next
``Context.sync()``.
"""
import ctypes
import struct

import numpy as np

from ._lib import PagedKVView, SeqBatchView, check, lib
from .ops import DeviceBuffer

F16, BF16, F32 = 0, 1, 2          # ALM_F16, ALM_BF16, ALM_F32
I32, F64 = "int32", "float64"
# type codes by the spellings of torch dtypes, numpy dtypes and array-interface type strings
_NAMES = {"float16": F16, "bfloat16": BF16, "float32": F32, "int32": I32, "float64": F64,
          "<f2": F16, "<f4": F32, "<i4": I32, "<f8": F64}
_CODES = {}                       # dtype object -> code
_SIZES = {F16: 2, BF16: 2, F32: 4, I32: 4, F64: 8}


class _Device:
    type = "cuda"

    def __init__(self, index):
        self.index = index


class DeviceArray:
    """A typed, shaped view of device memory of the library (``buf``: an
    ``ops.DeviceBuffer``; ``offset`` in bytes; contiguous)."""

    def __init__(self, buf, shape, dtype, offset=0):
        self.buf, self.shape, self.dtype, self.offset = buf, tuple(int(n) for n in shape), dtype, int(offset)
        size = _SIZES[_code(dtype)]
        if self.offset < 0 or self.offset + int(np.prod(self.shape, dtype=np.int64)) * size > buf.nbytes:
            raise ValueError("the view ends behind its buffer")

    @property
    def device(self):
        return _Device(self.buf.ctx.device)

    def data_ptr(self):
        return self.buf.h.value + self.offset

    def stride(self):
        out, n = [], 1
        for d in reversed(self.shape):
            out.append(n)
            n *= d
        return tuple(reversed(out))


def _code(dtype):
    try:
        return _CODES[dtype]
    except (KeyError, TypeError):
        pass
    name = dtype if isinstance(dtype, str) else str(dtype)
    code = _NAMES.get(name.replace("torch.", ""))
    if code is None and not isinstance(dtype, str):
        try:
            code = _NAMES.get(np.dtype(dtype).name)
        except TypeError:
            pass
    if code is None:
        raise TypeError(f"unsupported element type {name}")
    try:
        _CODES[dtype] = code
    except TypeError:
        pass
    return code


def _array(a, what, codes, ndim, device=None):
    """(pointer, type code, shape, strides in elements) of a device array."""
    if hasattr(a, "data_ptr"):
        dev = getattr(a, "device", None)
        if dev is not None:
            if getattr(dev, "type", "cuda") != "cuda":
                raise ValueError(f"{what} must be on a CUDA device")
            if device is not None and dev.index is not None and dev.index != device:
                raise ValueError(f"{what} is on device {dev.index}, not on device {device}")
        p, shape, stride, code = a.data_ptr(), a.shape, a.stride(), _code(a.dtype)
    elif hasattr(a, "__cuda_array_interface__"):
        i = a.__cuda_array_interface__
        p, shape, code = i["data"][0], tuple(i["shape"]), _code(i["typestr"])
        size = _SIZES[code]
        if i.get("strides") is None:
            stride, n = [], 1
            for d in reversed(shape):
                stride.append(n)
                n *= d
            stride = tuple(reversed(stride))
        else:
            if any(s % size for s in i["strides"]):
                raise ValueError(f"{what} has strides that are not whole elements")
            stride = tuple(s // size for s in i["strides"])
    else:
        raise TypeError(f"{what} must be a device array (data_ptr() or __cuda_array_interface__)")
    if code not in codes:
        raise TypeError(f"{what} has an unsupported element type")
    if len(shape) != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions")
    return p, code, shape, stride


def _dense(shape, stride):
    n = 1
    for d, s in zip(reversed(shape), reversed(stride)):
        if d != 1 and s != n:
            return 0 in shape
        n *= d
    return True


def _contiguous(a, what, codes, ndim, device=None):
    p, code, shape, stride = _array(a, what, codes, ndim, device)
    if not _dense(shape, stride):
        raise ValueError(f"{what} must be contiguous")
    return p, code, shape


def _flat(a, what, code, shape, device):
    """Pointer of a contiguous array of this type and shape.  (The first lines
    are the common case, a tensor that is all of that: these calls are made
    for every layer, and a launch takes a few microseconds.)"""
    try:
        if a.shape == shape and _CODES.get(a.dtype) == code and a.get_device() == device and a.is_contiguous():
            return a.data_ptr()
    except AttributeError:
        pass
    p, _, got, stride = _array(a, what, (code,), len(shape), device)
    if tuple(got) != shape:
        raise ValueError(f"{what} must be {shape}, not {tuple(got)}")
    if not _dense(shape, stride):
        raise ValueError(f"{what} must be contiguous")
    return p


def _rows(a, what, code, shape, device):
    """(pointer, row stride, head stride) of a (rows, heads, dim) array."""
    try:
        if a.shape == shape and _CODES.get(a.dtype) == code and a.get_device() == device:
            stride = a.stride()
            if stride[2] == 1 and shape[0] > 1 and shape[1] > 1:
                return a.data_ptr(), stride[0], stride[1]
    except AttributeError:
        pass
    p, _, got, stride = _array(a, what, (code,), 3, device)
    if tuple(got) != shape:
        raise ValueError(f"{what} must be {shape}, not {tuple(got)}")
    if stride[2] != 1 and shape[2] > 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    # a stride nothing is stepped with may be any number
    return p, stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0


def _on(ctx, *views):
    for v in views:
        if v.device is not None and v.device != ctx.device:
            raise ValueError(f"the {type(v).__name__} is on device {v.device}, the context on device {ctx.device}")


def _device_of(*arrays):
    """The device of the first array that tells one."""
    for a in arrays:
        index = getattr(getattr(a, "device", None), "index", None)
        if index is not None:
            return index
    return None


class PagedKV:
    """One layer's pages: K and V (n_pages, kv_heads, page_size, head_dim),
    contiguous, fp16 or bf16.  ``DeviceKV.view(layer)`` gives a model's own."""

    def __init__(self, k, v, device=None):
        self.device = device = _device_of(k, v) if device is None else device
        kp, code, shape = _contiguous(k, "k", (F16, BF16), 4, device)
        vp, vcode, vshape = _contiguous(v, "v", (F16, BF16), 4, device)
        if vcode != code or tuple(vshape) != tuple(shape):
            raise ValueError("k and v must have the same type and shape")
        self.code = code
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = (int(n) for n in shape)
        self.c = PagedKVView(kp, vp, code, self.n_pages, self.page_size, self.kv_heads, self.head_dim)
        self.ref = ctypes.addressof(self.c)
        self._keep = (k, v)

    @classmethod
    def of_view(cls, view, keep):
        self = cls.__new__(cls)
        self.code = view.dtype
        self.n_pages, self.kv_heads = view.n_pages, view.kv_heads
        self.page_size, self.head_dim = view.page_size, view.head_dim
        self.c, self._keep = view, keep
        self.ref = ctypes.addressof(view)
        self.device = keep.model.ctx.device
        return self


class PageTable:
    """The page table of a model's cache (``DeviceKV.page_table()``): row s
    holds slot s's page numbers."""

    def __init__(self, pointer, rows, pages, keep, device=None):
        self.pointer, self.rows, self.pages, self._keep, self.device = pointer, rows, pages, keep, _Device(device)


class SeqBatch:
    """The sequences of one pass.  ``row_start`` (n_seq + 1, int32): sequence
    s owns rows row_start[s] .. row_start[s + 1] - 1 of the packed row tensors;
    they are the last of its ``kv_len[s]`` (int32) positions.  ``page_table``
    (int32, a row per sequence, or per slot with ``slots``; or a
    ``PageTable``): position p lies on page page_table[s][p // page_size].
    ``n_rows``: rows of the packed tensors (rows behind the last sequence stay
    as they are).  ``max_rows`` bounds the rows of one sequence; it chooses
    the attention kernel.  All arrays stay on the device, so a captured pass
    can be replayed with new contents."""

    def __init__(self, row_start, kv_len, page_table, n_rows, max_rows=None, slots=None, device=None):
        self.device = device = _device_of(row_start, kv_len, page_table, slots) if device is None else device
        rp, _, rs = _contiguous(row_start, "row_start", (I32,), 1, device)
        lp, _, ls = _contiguous(kv_len, "kv_len", (I32,), 1, device)
        n_seq = int(ls[0])
        if rs[0] != n_seq + 1:
            raise ValueError("row_start must have one entry more than kv_len")
        if isinstance(page_table, PageTable):
            if page_table.device.index not in (None, device):
                raise ValueError(f"page_table is on device {page_table.device.index}, not on device {device}")
            tp, rows, pages, step = page_table.pointer, page_table.rows, page_table.pages, page_table.pages
        else:
            tp, _, shape, stride = _array(page_table, "page_table", (I32,), 2, device)
            rows, pages = int(shape[0]), int(shape[1])
            if pages > 1 and stride[1] != 1:
                raise ValueError("page_table must be contiguous in its last dimension")
            step = int(stride[0]) if rows > 1 else pages
            if step < pages:
                raise ValueError("page_table rows must not overlap")
            if step > _INT_MAX:
                raise ValueError("page_table rows must lie less than 2^31 elements apart")
        sp = None
        if slots is not None:
            sp, _, ss = _contiguous(slots, "slots", (I32,), 1, device)
            if ss[0] != n_seq:
                raise ValueError("slots must have an entry for every sequence")
        elif rows < n_seq:
            raise ValueError("page_table must have a row for every sequence")
        self.n_seq, self.n_rows = n_seq, int(n_rows)
        if not 0 <= self.n_rows <= _INT_MAX:
            raise ValueError("n_rows must not be negative and be below 2^31")
        most = self.n_rows if max_rows is None else min(int(max_rows), _INT_MAX)
        self.c = SeqBatchView(n_seq, self.n_rows, most, rows, pages, step, rp, lp, tp, sp)
        self.ref = ctypes.addressof(self.c)
        self._keep = (row_start, kv_len, page_table, slots)


class AttnWorkspace:
    """Work area of ``attn_paged`` (partial results of sequences that several
    CTAs share, counters of those that are ready), for any batch of these heads.  Calls that can overlap on the
    GPU, graphs replayed on different streams among them, need one each."""

    def __init__(self, ctx, heads, kv_heads, head_dim):
        n = ctypes.c_size_t()
        check(lib.alm_attn_paged_work(ctx.h, int(heads), int(kv_heads), int(head_dim), ctypes.byref(n)))
        self.buf = DeviceBuffer(ctx, n.value)
        self.buf.upload(np.zeros(min(n.value, 1 << 16), np.uint8))   # the counters at its start
        self.pointer, self.nbytes, self.device = self.buf.h.value, n.value, ctx.device


# The argument structs of the header, packed at once (native alignment).
_ROPE_ARGS = struct.Struct("@PPPqqqqqqPqqiPPfPiiii").pack
_ATTN_ARGS = struct.Struct("@PqqPqqPqiifPN").pack
_VERIFY_ARGS = struct.Struct("@iiiiPPiqPPqqPPPPPP").pack
_INT_MAX = 2 ** 31 - 1


def _packed(pack, what, *args):
    try:
        return pack(*args)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"{what}: an argument is no number of its type ({e})") from None


def _heads_of(q, what, n_rows, dim):
    """(n_rows, heads, dim) with q's own number of heads."""
    shape = getattr(q, "shape", None)
    if shape is None:
        shape = _array(q, what, (F16, BF16), 3)[2]
    if len(shape) != 3:
        raise ValueError(f"{what} must have 3 dimensions")
    return n_rows, int(shape[1]), dim


def rope_append(ctx, kv, seqs, q, k, v, rope, q_out, q_norm=None, k_norm=None, eps=1e-6, interleaved=False):
    """alm_rope_append: norm (optional) and rotate the heads of q and k, write
    q to ``q_out`` and K / V to the cache.  q, q_out (n_rows, heads, head_dim),
    k, v (n_rows, kv_heads, head_dim): the cache's type, any row and head
    strides that are multiples of 8; q_out may be q.  rope (positions,
    rot_dim): [cos | sin], fp16, bf16 or fp32; interleaved rotates neighbours
    (2i, 2i + 1) instead of halves (i, i + rot_dim / 2)."""
    dev, n, d, code, hk = ctx.device, seqs.n_rows, kv.head_dim, kv.code, kv.kv_heads
    if kv.device != dev or seqs.device != dev:
        _on(ctx, kv, seqs)
    shape = _heads_of(q, "q", n, d)
    qp, qr, qh = _rows(q, "q", code, shape, dev)
    op, o_r, oh = _rows(q_out, "q_out", code, shape, dev)
    heads, shape = shape[1], (n, hk, d)
    kp, kr, kh = _rows(k, "k", code, shape, dev)
    vp, vr, vh = _rows(v, "v", code, shape, dev)
    rp, rcode, rs = _contiguous(rope, "rope", (F16, BF16, F32), 2, dev)
    qw = _flat(q_norm, "q_norm", code, (d,), dev) if q_norm is not None else 0
    kw = _flat(k_norm, "k_norm", code, (d,), dev) if k_norm is not None else 0
    check(lib.alm_rope_append(ctx.h, kv.ref, seqs.ref, _packed(
        _ROPE_ARGS, "rope_append", qp, kp, vp, qr, qh, kr, kh, vr, vh, op, o_r, oh, heads, qw, kw, eps, rp, rcode,
        rs[0], rs[1], 1 if interleaved else 0)))


def attn_paged(ctx, kv, seqs, q, out, work, scale=None, window=0, lse=None):
    """alm_attn_paged: out[r] = softmax(scale q[r] . K) V over the positions of
    row r's sequence up to its own (the last ``window`` of them when window >
    0).  q, out (n_rows, heads, head_dim) of the cache's type, not the same
    memory; scale defaults to head_dim ** -0.5; lse (n_rows, heads) fp32
    receives the log of the sum of exponentials.  Rows that see nothing get
    zeros and -inf."""
    dev, n, d, code = ctx.device, seqs.n_rows, kv.head_dim, kv.code
    if kv.device != dev or seqs.device != dev or work.device != dev:
        _on(ctx, kv, seqs, work)
    shape = _heads_of(q, "q", n, d)
    qp, qr, qh = _rows(q, "q", code, shape, dev)
    op, o_r, oh = _rows(out, "out", code, shape, dev)
    lp, ls = 0, 0
    if lse is not None:
        lp, _, got, stride = _array(lse, "lse", (F32,), 2, dev)
        if tuple(got) != shape[:2] or (shape[1] > 1 and stride[1] != 1):
            raise ValueError("lse must be (n_rows, heads), contiguous in its last dimension")
        ls = stride[0]
    check(lib.alm_attn_paged(ctx.h, kv.ref, seqs.ref, _packed(
        _ATTN_ARGS, "attn_paged", qp, qr, qh, op, o_r, oh, lp, ls, shape[1], window,
        d ** -0.5 if scale is None else scale, work.pointer, work.nbytes)))


def verify(ctx, row_start, logits, draft_tokens, draft_probs, uniforms, temperature, tokens, n_accepted,
           min_p=None, p_draft=None):
    """alm_verify: accept drafted tokens while u q(x) < p(x), then draw from
    the residual (or the bonus row), for a ragged batch.  row_start (n_seq + 1,
    int32): sequence s owns rows row_start[s] .. row_start[s + 1] - 1 of logits
    (n_rows, vocab): one per drafted token and one more.  draft_tokens (n_seq,
    k_max) int32; draft_probs (n_seq, k_max, vocab) fp32 or None (certain
    drafts); uniforms (n_seq, k_max + 1) float64; temperature, min_p (n_seq)
    fp32, temperature <= 0 greedy.  Writes tokens (n_seq, k_max + 1) int32 (-1
    behind the emitted ones), n_accepted (n_seq) int32 and p_draft (n_seq,
    k_max) fp32."""
    dev = ctx.device
    lp, lcode, ls, lstride = _array(logits, "logits", (F16, BF16, F32), 2, dev)
    n_rows, vocab = ls
    if vocab > 1 and lstride[1] != 1:
        raise ValueError("logits must be contiguous in the last dimension")
    dp, _, ds = _contiguous(draft_tokens, "draft_tokens", (I32,), 2, dev)
    n_seq, k = ds
    rp = _flat(row_start, "row_start", I32, (n_seq + 1,), dev)
    qp, q_seq, q_step = 0, 0, 0
    if draft_probs is not None:
        qp, _, qs, qst = _array(draft_probs, "draft_probs", (F32,), 3, dev)
        if tuple(qs) != (n_seq, k, vocab) or (vocab > 1 and qst[2] != 1):
            raise ValueError("draft_probs must be (n_seq, k_max, vocab), contiguous in its last dimension")
        q_seq, q_step = qst[0], qst[1]
    up = _flat(uniforms, "uniforms", F64, (n_seq, k + 1), dev)
    op = _flat(tokens, "tokens", I32, (n_seq, k + 1), dev)
    tp = _flat(temperature, "temperature", F32, (n_seq,), dev)
    ap = _flat(n_accepted, "n_accepted", I32, (n_seq,), dev)
    mp = _flat(min_p, "min_p", F32, (n_seq,), dev) if min_p is not None else 0
    pp = _flat(p_draft, "p_draft", F32, (n_seq, k), dev) if p_draft is not None else 0
    check(lib.alm_verify(ctx.h, _packed(
        _VERIFY_ARGS, "verify", n_seq, n_rows, k, vocab, rp, lp, lcode, lstride[0] if n_rows > 1 else vocab, dp, qp,
        q_seq, q_step, up, tp, mp, op, ap, pp)))
