"""Refusals of the operators on device data (paged.py and its C entries).
Arguments are checked before the context, so every refusal shows without a
GPU; the pointers are made up and never followed."""
import ctypes

import numpy as np
import pytest

from androidllm_b200 import paged
from androidllm_b200._lib import AttnPagedArgs, PagedKVView, RopeAppendArgs, SeqBatchView, VerifyArgs, lib

P = 1 << 20      # an aligned address


class Fake:
    """A device array that exists in name only."""

    def __init__(self, shape, dtype="float16", stride=None, ptr=P, device=None):
        self.shape, self.dtype, self._ptr = tuple(shape), dtype, ptr
        st, n = [], 1
        for d in reversed(self.shape):
            st.append(n)
            n *= d
        self._stride = tuple(reversed(st)) if stride is None else stride
        if device is not None:
            self.device = device

    def data_ptr(self):
        return self._ptr

    def stride(self):
        return self._stride


class NoContext:
    h, device = None, 0


def _kv(**kw):
    a = dict(k_dev=P, v_dev=P, dtype=0, n_pages=4, page_size=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return PagedKVView(**a)


def _batch(**kw):
    a = dict(n_seq=2, n_rows=5, max_rows=3, table_rows=2, table_pages=4, page_stride=4, row_start_dev=P, kv_len_dev=P,
             page_table_dev=P, slots_dev=None)
    a.update(kw)
    return SeqBatchView(**a)


def _rope(**kw):
    a = dict(q_dev=P, k_dev=P, v_dev=P, q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, q_out_dev=P,
             qo_row=256, qo_head=64, heads=4, eps=1e-6, rope_dev=P, rope_dtype=0, rope_rows=64, rot_dim=64,
             interleaved=0)
    a.update(kw)
    return RopeAppendArgs(**a)


def _attn(**kw):
    a = dict(q_dev=P, q_row=256, q_head=64, out_dev=P, out_row=256, out_head=64, lse_dev=None, lse_row=4, heads=4,
             window=0, scale=0.125, work_dev=P, work_bytes=1 << 40)
    a.update(kw)
    return AttnPagedArgs(**a)


def _verify(**kw):
    a = dict(n_seq=2, n_rows=6, k_max=3, vocab=100, row_start_dev=P, logits_dev=P, logits_dtype=0, logits_row=100,
             draft_tokens_dev=P, draft_probs_dev=None, q_seq=0, q_step=0, uniforms_dev=P, temperature_dev=P,
             min_p_dev=None, tokens_dev=P, n_accepted_dev=P, p_draft_dev=None)
    a.update(kw)
    return VerifyArgs(**a)


def _refused(rc, word):
    assert rc == 1
    msg = lib.alm_last_error().decode()
    assert word in msg, msg


def _ref(c):
    return ctypes.byref(c)


BAD_KV = [(dict(k_dev=None), "null"), (dict(dtype=2), "fp16 or bf16"), (dict(dtype=-1), "fp16 or bf16"),
          (dict(head_dim=48), "head_dim"), (dict(head_dim=512), "head_dim"), (dict(kv_heads=0), "kv_heads"),
          (dict(n_pages=0), "page"), (dict(page_size=0), "page_size"), (dict(page_size=70000), "page_size"),
          (dict(v_dev=P + 8), "aligned")]
BAD_BATCH = [(dict(n_seq=-1), "n_seq"), (dict(n_seq=4097, table_rows=5000), "n_seq"), (dict(n_rows=-1), "n_rows"),
             (dict(max_rows=-1), "max_rows"), (dict(kv_len_dev=None), "null"), (dict(table_rows=1), "page table"),
             (dict(slots_dev=P, table_rows=0), "page table"), (dict(page_stride=3), "page_stride"),
             (dict(row_start_dev=P + 2), "aligned"), (dict(page_table_dev=P + 1), "aligned"),
             (dict(slots_dev=P + 2), "aligned")]


@pytest.mark.parametrize("kw,word", BAD_KV)
def test_cache_refusals(kw, word):
    _refused(lib.alm_rope_append(None, _ref(_kv(**kw)), _ref(_batch()), _ref(_rope())), word)
    _refused(lib.alm_attn_paged(None, _ref(_kv(**kw)), _ref(_batch()), _ref(_attn())), word)


@pytest.mark.parametrize("kw,word", BAD_BATCH)
def test_batch_refusals(kw, word):
    _refused(lib.alm_rope_append(None, _ref(_kv()), _ref(_batch(**kw)), _ref(_rope())), word)
    _refused(lib.alm_attn_paged(None, _ref(_kv()), _ref(_batch(**kw)), _ref(_attn())), word)


@pytest.mark.parametrize("kw,word", [
    (dict(heads=0), "heads"), (dict(q_dev=None), "null"), (dict(rope_dev=None), "null"), (dict(q_dev=P + 2), "aligned"),
    (dict(q_norm_dev=P + 4), "aligned"), (dict(q_row=257), "stride"), (dict(v_head=68), "stride"),
    (dict(rope_dtype=3), "table"), (dict(rope_rows=0), "table"), (dict(rot_dim=8), "rot_dim"),
    (dict(rot_dim=72), "rot_dim"), (dict(rot_dim=128), "rot_dim"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), ({}, "null ctx")])
def test_append_refusals(kw, word):
    _refused(lib.alm_rope_append(None, _ref(_kv()), _ref(_batch()), _ref(_rope(**kw))), word)


@pytest.mark.parametrize("kw,word", [
    (dict(heads=0), "heads"), (dict(heads=5), "multiple"), (dict(heads=258), "128"), (dict(out_dev=None), "null"),
    (dict(work_dev=None), "null"), (dict(q_dev=P + 8), "aligned"), (dict(out_head=65), "stride"),
    (dict(window=-1), "window"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=2e30), "scale"), (dict(scale=float("nan")), "scale"), (dict(work_dev=P + 128), "256-byte"),
    (dict(lse_dev=P + 2), "aligned"), ({}, "null ctx")])
def test_attention_refusals(kw, word):
    _refused(lib.alm_attn_paged(None, _ref(_kv()), _ref(_batch()), _ref(_attn(**kw))), word)


@pytest.mark.parametrize("kw,word", [
    (dict(n_seq=-1), "n_seq"), (dict(n_rows=-1), "n_rows"), (dict(k_max=32), "k_max"), (dict(k_max=-1), "k_max"),
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1), "vocab"), (dict(logits_dtype=7), "type"),
    (dict(row_start_dev=None), "null"), (dict(logits_dev=None), "null"), (dict(draft_tokens_dev=None), "null"),
    (dict(uniforms_dev=None), "null"), (dict(temperature_dev=None), "null"), (dict(logits_row=99), "logits_row"),
    (dict(logits_dev=P + 1), "aligned"), (dict(uniforms_dev=P + 4), "aligned"), (dict(draft_probs_dev=P + 2), "aligned"),
    (dict(tokens_dev=P + 2), "aligned"), ({}, "null ctx")])
def test_verify_refusals(kw, word):
    _refused(lib.alm_verify(None, _ref(_verify(**kw))), word)


def test_null_structs():
    _refused(lib.alm_rope_append(None, None, _ref(_batch()), _ref(_rope())), "null")
    _refused(lib.alm_rope_append(None, _ref(_kv()), None, _ref(_rope())), "null")
    _refused(lib.alm_attn_paged(None, _ref(_kv()), _ref(_batch()), None), "null")
    _refused(lib.alm_verify(None, None), "null")
    _refused(lib.alm_attn_paged_work(None, 4, 2, 64, None), "null")
    n = ctypes.c_size_t()
    _refused(lib.alm_attn_paged_work(None, 5, 2, 64, ctypes.byref(n)), "multiple")
    _refused(lib.alm_kv_view(None, 0, None, None, None, None), "null")
    _refused(lib.alm_ctx_create_on_stream(0, None, None), "null")


def _seqs(**kw):
    a = dict(row_start=Fake((3,), "int32"), kv_len=Fake((2,), "int32"), page_table=Fake((2, 4), "int32"), n_rows=5)
    a.update(kw)
    return paged.SeqBatch(**a)


def _cache():
    return paged.PagedKV(Fake((4, 2, 16, 64)), Fake((4, 2, 16, 64)))


class Cpu:
    type, index = "cpu", None


class Gpu1:
    type, index = "cuda", 1


@pytest.mark.parametrize("make,err", [
    (lambda: paged.PagedKV(Fake((4, 2, 16, 64)), Fake((4, 2, 16, 64), "bfloat16")), ValueError),
    (lambda: paged.PagedKV(Fake((4, 2, 16, 64)), Fake((4, 2, 16, 32))), ValueError),
    (lambda: paged.PagedKV(Fake((4, 2, 16, 64), "float32"), Fake((4, 2, 16, 64), "float32")), TypeError),
    (lambda: paged.PagedKV(Fake((2, 16, 64)), Fake((2, 16, 64))), ValueError),
    (lambda: paged.PagedKV(Fake((4, 2, 16, 64), stride=(4096, 1024, 128, 1)), Fake((4, 2, 16, 64))), ValueError),
    (lambda: paged.PagedKV(np.zeros((4, 2, 16, 64), np.float16), np.zeros((4, 2, 16, 64), np.float16)), TypeError),
    (lambda: paged.PagedKV(Fake((4, 2, 16, 64), device=Cpu), Fake((4, 2, 16, 64))), ValueError),
    (lambda: _seqs(row_start=Fake((2,), "int32")), ValueError),
    (lambda: _seqs(row_start=Fake((3,), "float32")), TypeError),
    (lambda: _seqs(page_table=Fake((1, 4), "int32")), ValueError),
    (lambda: _seqs(page_table=Fake((2, 4), "int32", stride=(1, 2))), ValueError),
    (lambda: _seqs(page_table=Fake((2, 4), "int32", stride=(2, 1))), ValueError),
    (lambda: _seqs(slots=Fake((3,), "int32")), ValueError),
    (lambda: _seqs(n_rows=-1), ValueError),
])
def test_python_views_refuse(make, err):
    with pytest.raises(err):
        make()


@pytest.mark.parametrize("kw,err", [
    (dict(q=Fake((5, 4, 32))), ValueError), (dict(q=Fake((4, 4, 64))), ValueError),
    (dict(q=Fake((5, 4, 64), "bfloat16")), TypeError), (dict(k=Fake((5, 3, 64))), ValueError),
    (dict(q_out=Fake((5, 3, 64))), ValueError), (dict(rope=Fake((9, 64), "int32")), TypeError),
    (dict(rope=Fake((9, 64), stride=(128, 1))), ValueError), (dict(q_norm=Fake((32,))), ValueError),
    (dict(q=Fake((5, 4, 64), stride=(256, 64, 2))), ValueError), (dict(q=Fake((5, 4, 64), device=Gpu1)), ValueError)])
def test_python_append_refuses(kw, err):
    a = dict(q=Fake((5, 4, 64)), k=Fake((5, 2, 64)), v=Fake((5, 2, 64)), rope=Fake((9, 64)), q_out=Fake((5, 4, 64)))
    a.update(kw)
    with pytest.raises(err):
        paged.rope_append(NoContext, _cache(), _seqs(), **a)


@pytest.mark.parametrize("kw,err", [
    (dict(out=Fake((5, 3, 64))), ValueError), (dict(lse=Fake((5, 3), "float32")), ValueError),
    (dict(lse=Fake((5, 4))), TypeError), (dict(out=Fake((5, 4, 64), "float32")), TypeError)])
def test_python_attention_refuses(kw, err):
    class Work:
        pointer, nbytes, device = P, 1 << 30, None
    a = dict(q=Fake((5, 4, 64)), out=Fake((5, 4, 64)), work=Work)
    a.update(kw)
    with pytest.raises(err):
        paged.attn_paged(NoContext, _cache(), _seqs(), **a)


@pytest.mark.parametrize("kw,err", [
    (dict(row_start=Fake((2,), "int32")), ValueError), (dict(uniforms=Fake((2, 4), "float32")), TypeError),
    (dict(uniforms=Fake((2, 3), "float64")), ValueError), (dict(tokens=Fake((2, 3), "int32")), ValueError),
    (dict(draft_probs=Fake((2, 3, 99), "float32")), ValueError), (dict(temperature=Fake((3,), "float32")), ValueError),
    (dict(min_p=Fake((1,), "float32")), ValueError), (dict(p_draft=Fake((2, 4), "float32")), ValueError),
    (dict(logits=Fake((6, 100), "float64")), TypeError), (dict(n_accepted=Fake((3,), "int32")), ValueError)])
def test_python_verify_refuses(kw, err):
    a = dict(row_start=Fake((3,), "int32"), logits=Fake((6, 100)), draft_tokens=Fake((2, 3), "int32"),
             draft_probs=None, uniforms=Fake((2, 4), "float64"), temperature=Fake((2,), "float32"),
             tokens=Fake((2, 4), "int32"), n_accepted=Fake((2,), "int32"))
    a.update(kw)
    with pytest.raises(err):
        paged.verify(NoContext, **a)


@pytest.mark.parametrize("args,pack", [
    (RopeAppendArgs, paged._ROPE_ARGS), (AttnPagedArgs, paged._ATTN_ARGS), (VerifyArgs, paged._VERIFY_ARGS)])
def test_packed_arguments_are_the_structs(args, pack):
    """The calls' packed bytes fill the header's structs field by field."""
    vals = [i + 1 if t is not ctypes.c_float else 0.5 * (i + 1) for i, (_, t) in enumerate(args._fields_)]
    raw = pack(*vals)
    assert len(raw) == ctypes.sizeof(args)
    got = args.from_buffer_copy(raw)
    assert [getattr(got, n) for n, _ in args._fields_] == vals


def test_empty_arrays_are_contiguous():
    assert paged._dense((2, 0), (1, 1)) and paged._dense((0, 5), (7, 1)) and not paged._dense((2, 3), (4, 1))


class Gpu0:
    type, index = "cuda", 0


class Buffer:
    """Memory of a context, in name only."""

    def __init__(self, device):
        class Ctx:
            pass

        class Handle:
            value = P
        self.ctx, self.h, self.nbytes = Ctx(), Handle(), 1 << 20
        self.ctx.device = device


@pytest.mark.parametrize("make", [
    lambda: paged.PagedKV(Fake((4, 2, 16, 64), device=Gpu0), Fake((4, 2, 16, 64), device=Gpu1)),
    lambda: _seqs(row_start=Fake((3,), "int32", device=Gpu0), kv_len=Fake((2,), "int32", device=Gpu1)),
    lambda: _seqs(row_start=Fake((3,), "int32", device=Gpu0), page_table=Fake((2, 4), "int32", device=Gpu1)),
    lambda: _seqs(row_start=Fake((3,), "int32", device=Gpu1), slots=Fake((2,), "int32", device=Gpu0)),
    lambda: _seqs(row_start=Fake((3,), "int32", device=Gpu0), page_table=paged.PageTable(P, 2, 4, None, device=1)),
    lambda: _seqs(row_start=Fake((3,), "int32", device=Gpu0), kv_len=paged.DeviceArray(Buffer(1), (2,), "int32")),
    lambda: paged.PagedKV(paged.DeviceArray(Buffer(0), (1, 2, 16, 64), "float16"), Fake((1, 2, 16, 64), device=Gpu1)),
])
def test_views_refuse_arrays_of_different_devices(make):
    with pytest.raises(ValueError, match="device"):
        make()


def test_views_know_their_device():
    kv = paged.PagedKV(Fake((4, 2, 16, 64)), Fake((4, 2, 16, 64), device=Gpu1))
    assert kv.device == 1
    assert paged.PagedKV(*[paged.DeviceArray(Buffer(1), (1, 2, 16, 64), "float16")] * 2).device == 1
    seqs = _seqs(page_table=paged.PageTable(P, 2, 4, None, device=1))
    assert seqs.device == 1
    with pytest.raises(ValueError, match="device"):      # NoContext is on device 0
        paged.rope_append(NoContext, kv, _seqs(), Fake((5, 4, 64)), Fake((5, 2, 64)), Fake((5, 2, 64)), Fake((9, 64)),
                          Fake((5, 4, 64)))
    with pytest.raises(ValueError, match="device"):
        paged.rope_append(NoContext, _cache(), seqs, Fake((5, 4, 64)), Fake((5, 2, 64)), Fake((5, 2, 64)), Fake((9, 64)),
                          Fake((5, 4, 64)))


@pytest.mark.parametrize("kw", [dict(window=2 ** 31), dict(window=-2 ** 40), dict(window=1.5)])
def test_python_attention_refuses_numbers_outside_their_types(kw):
    class Work:
        pointer, nbytes, device = P, 1 << 30, None
    with pytest.raises(ValueError, match="attn_paged"):
        paged.attn_paged(NoContext, _cache(), _seqs(), Fake((5, 4, 64)), Fake((5, 4, 64)), Work, **kw)


def test_python_refuses_floats_outside_their_type():
    from androidllm_b200._lib import ALMError

    class Work:
        pointer, nbytes, device = P, 1 << 30, None
    with pytest.raises(ALMError, match="scale"):         # an infinity in 32 bits
        paged.attn_paged(NoContext, _cache(), _seqs(), Fake((5, 4, 64)), Fake((5, 4, 64)), Work, scale=1e60)
    with pytest.raises(ALMError, match="eps"):
        paged.rope_append(NoContext, _cache(), _seqs(), Fake((5, 4, 64)), Fake((5, 2, 64)), Fake((5, 2, 64)),
                          Fake((9, 64)), Fake((5, 4, 64)), eps=1e60)


def test_batches_refuse_or_clamp_numbers_outside_their_types():
    with pytest.raises(ValueError, match="page_table"):
        _seqs(page_table=Fake((2, 4), "int32", stride=(2 ** 31, 1)))
    with pytest.raises(ValueError, match="n_rows"):
        _seqs(n_rows=2 ** 32 + 5)
    assert _seqs(max_rows=2 ** 40).c.max_rows == 2 ** 31 - 1       # a bound, and this one holds too
