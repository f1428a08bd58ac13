"""Refusals of the cache, attention and log-probability entry points, without a GPU: every check stands in front of the first CUDA
call, so a context of zeros is enough to reach it. And the 64-bit reference of the GPU tests against itself."""
import ctypes

from types import SimpleNamespace

import numpy as np
import pytest

from nn_b200 import _lib, api
from nn_b200.kv_cache import KvBatch, KvCache, _Batch, _Cache
from tests import kv_reference as ref

P = 1 << 20   # a pointer that nothing follows: aligned, not NULL
INVALID, SHAPE, UNSUPPORTED, RANGE = 1, 4, 10, 11


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture
def ctx():
    return ctypes.create_string_buffer(8192)


def cache(**kw):
    c = dict(format=0, kv_heads=2, dim=128, block=16, blocks=10, k=P, v=P, k_exp=P, v_exp=P)
    c.update(kw)
    return _Cache(**c)


BAD_CACHES = [(dict(format=2), INVALID), (dict(format=-1), INVALID), (dict(dim=96), UNSUPPORTED), (dict(dim=512), UNSUPPORTED), (dict(dim=0), UNSUPPORTED),
              (dict(block=8), UNSUPPORTED), (dict(block=24), UNSUPPORTED), (dict(block=512), UNSUPPORTED), (dict(block=-16), UNSUPPORTED), (dict(kv_heads=0), INVALID),
              (dict(kv_heads=70000), INVALID), (dict(blocks=0), INVALID), (dict(blocks=1 << 27), UNSUPPORTED), (dict(k=None), INVALID), (dict(v_exp=None), INVALID),
              (dict(v=P + 8), INVALID)]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_caches_that_are_refused(lib, ctx, kw, status):
    c = cache(**kw)
    b = _Batch(P, P, P, 1, 4, 1, 1)
    need = ctypes.c_size_t()
    assert lib.nnq_kv_append(ctx, ctypes.byref(c), P, 1 << 16, P, 1 << 16, 0, P, 1, None) == status
    assert lib.nnq_kv_read(ctx, ctypes.byref(c), P, 1, P, P, 0, None) == status
    assert lib.nnq_kv_attention_workspace(ctx, ctypes.byref(c), ctypes.byref(b), 140000, ctypes.byref(need)) == status
    assert lib.nnq_last_error(ctx)


@pytest.mark.parametrize("change,status", [
    (dict(requests=0), INVALID), (dict(n_free=-1), INVALID), (dict(table_ld=0), INVALID), (dict(rows=-1), INVALID), (dict(rows=1 << 31), UNSUPPORTED),
    (dict(requests=1 << 30), UNSUPPORTED), (dict(block=48), UNSUPPORTED), (dict(past=None), INVALID), (dict(count=None), INVALID), (dict(free=None), INVALID),
    (dict(table=None), INVALID), (dict(length=None), INVALID), (dict(row_start=None), INVALID), (dict(slot=None), INVALID), (dict(position=None), INVALID)])
def test_tables_that_are_refused(lib, ctx, change, status):
    a = dict(past=P, count=P, requests=2, free=P, n_free=4, skip=None, block=16, table=P, table_ld=4, length=P, row_start=P, slot=P, position=P, rows=2, used=None)
    a.update(change)
    assert lib.nnq_kv_tables(ctx, *a.values(), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dt=2), INVALID), (dict(rows=-1), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(slot=None), INVALID), (dict(k_ld=255), SHAPE),
    (dict(v_ld=128), SHAPE), (dict(k_ld=257), INVALID), (dict(k=P + 4), INVALID), (dict(v=P + 2), INVALID)])
def test_appends_that_are_refused(lib, ctx, change, status):
    a = dict(k=P, k_ld=256, v=P, v_ld=256, dt=0, slot=P, rows=3)
    a.update(change)
    assert lib.nnq_kv_append(ctx, ctypes.byref(cache()), *a.values(), None) == status


@pytest.mark.parametrize("change,status", [(dict(rows=-1), INVALID), (dict(slot=None), INVALID), (dict(k=None), INVALID), (dict(v=P + 4), INVALID), (dict(dt=5), INVALID)])
def test_reads_that_are_refused(lib, ctx, change, status):
    a = dict(slot=P, rows=3, k=P, v=P, dt=0)
    a.update(change)
    assert lib.nnq_kv_read(ctx, ctypes.byref(cache()), *a.values(), None) == status


@pytest.mark.parametrize("change,batch,status", [
    (dict(q_dt=3), {}, INVALID), (dict(y_dt=-1), {}, INVALID), (dict(heads=3), {}, SHAPE), (dict(heads=0), {}, SHAPE), (dict(scale=0.0), {}, RANGE),
    (dict(scale=-1.0), {}, RANGE), (dict(scale=float("nan")), {}, RANGE), (dict(scale=float("inf")), {}, RANGE), (dict(window=-1), {}, INVALID),
    (dict(q=None), {}, INVALID), (dict(y=None), {}, INVALID), (dict(q=P + 8), {}, INVALID), (dict(q_ld=511), {}, SHAPE), (dict(y_ld=513), {}, INVALID),
    (dict(work=None), {}, INVALID), (dict(work=P + 4), {}, INVALID), (dict(), dict(requests=0), INVALID), (dict(), dict(table_ld=0), INVALID), (dict(), dict(table_ld=1 << 27), UNSUPPORTED),
    (dict(), dict(rows=-1), INVALID), (dict(), dict(max_rows=0), INVALID), (dict(), dict(rows=1 << 30), UNSUPPORTED), (dict(), dict(length=None), INVALID),
    (dict(), dict(row_start=None), INVALID), (dict(), dict(table=None), INVALID)])
def test_attention_that_is_refused(lib, ctx, change, batch, status):
    b = dict(length=P, row_start=P, table=P, requests=1, table_ld=4, rows=2, max_rows=1)
    b.update(batch)
    a = dict(q=P, q_dt=0, q_ld=512, heads=4, scale=0.1, window=0, y=P, y_dt=0, y_ld=512, work=P, bytes=1 << 40)
    a.update(change)
    assert lib.nnq_kv_attention(ctx, ctypes.byref(cache()), ctypes.byref(_Batch(**b)), *a.values(), None) == status
    if status != INVALID or not change:
        assert lib.nnq_last_error(ctx)


def test_null_structures_are_refused(lib, ctx):
    need, b, c = ctypes.c_size_t(), _Batch(P, P, P, 1, 4, 1, 1), cache()
    assert lib.nnq_kv_append(ctx, None, P, 256, P, 256, 0, P, 1, None) == INVALID
    assert lib.nnq_kv_attention_workspace(ctx, ctypes.byref(c), None, 4, ctypes.byref(need)) == INVALID
    assert lib.nnq_kv_attention_workspace(ctx, ctypes.byref(c), ctypes.byref(b), 4, None) == INVALID
    for call in (lambda: lib.nnq_kv_tables(None, P, P, 1, P, 1, None, 16, P, 1, P, P, P, P, 1, None, None), lambda: lib.nnq_kv_read(None, None, P, 1, P, P, 0, None),
                 lambda: lib.nnq_token_logprobs(None, P, 0, 1, 8, 8, P, 0, P, P, P, P, None)):
        assert call() == INVALID


@pytest.mark.parametrize("change,status", [
    (dict(dt=2), INVALID), (dict(rows=-1), INVALID), (dict(vocab=0), INVALID), (dict(vocab=1 << 31), INVALID), (dict(ld=99), SHAPE), (dict(top=-1), UNSUPPORTED),
    (dict(top=33), UNSUPPORTED), (dict(vocab=5, top=6), UNSUPPORTED), (dict(x=None), INVALID), (dict(token=None), INVALID), (dict(x=P + 2), INVALID),
    (dict(tt=None, tl=None), INVALID), (dict(top=0, lp=None, ent=None), INVALID)])
def test_log_probabilities_that_are_refused(lib, ctx, change, status):
    a = dict(x=P, dt=0, rows=2, vocab=100, ld=100, token=P, top=4, lp=P, ent=P, tt=P, tl=P)
    a.update(change)
    assert lib.nnq_token_logprobs(ctx, *a.values(), None) == status


def test_calls_without_rows_do_nothing(lib, ctx):
    c, b = cache(), _Batch(P, P, P, 1, 4, 0, 1)
    assert lib.nnq_kv_append(ctx, ctypes.byref(c), None, 256, None, 256, 0, None, 0, None) == 0
    assert lib.nnq_kv_read(ctx, ctypes.byref(c), None, 0, None, None, 0, None) == 0
    assert lib.nnq_kv_attention(ctx, ctypes.byref(c), ctypes.byref(b), None, 0, 512, 4, 0.1, 0, None, 0, 512, None, 0, None) == 0
    assert lib.nnq_token_logprobs(ctx, None, 0, 0, 10, 10, None, 0, None, None, None, None, None) == 0


@pytest.mark.parametrize("fmt", [0, 1])
def test_the_reference_keeps_every_code(fmt):
    """Values of codes round to themselves, and a block's exponent is the least that holds its largest value."""
    v = ref.VALUES[fmt][np.abs(ref.VALUES[fmt]) <= ref.TOP[fmt]]
    assert np.array_equal(ref.round_code(fmt, v), v)
    for amax in (127.0, 127.5, 448.0, 448.5, 1.0, 3e-20, 2e38):
        e = ref.least_exponent(fmt, amax)
        assert amax <= ref.TOP[fmt] * 2.0 ** (e - 127) and (e == 7 or amax > ref.TOP[fmt] * 2.0 ** (e - 128))


class DeviceInts:
    """What a batch asks of an int32 tensor on the device, without one."""

    def __init__(self, *shape):
        torch = pytest.importorskip("torch")
        self.shape, self.dtype, self.is_cuda, self.device = torch.Size(shape), torch.int32, True, "cuda:0"

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True


@pytest.mark.parametrize("slots,positions", [(10, 5), (10, 0), (3, 4)])
def test_a_batch_has_a_position_for_every_slot(slots, positions):
    """`build` writes both for as many rows as there are slots."""
    with pytest.raises(api.ShapeMismatch):
        KvBatch.from_tensors(DeviceInts(2, 4), DeviceInts(2), DeviceInts(3), 16, slot=DeviceInts(slots), position=DeviceInts(positions), backend=SimpleNamespace(device=0))


@pytest.mark.parametrize("over,status", [(0, UNSUPPORTED), (1100, 0)])
def test_query_vectors_are_counted_in_32_bits(lib, ctx, over, status):
    """Up to an item of 256 vectors beyond the last, so the last thousand numbers of the range are left out."""
    need, heads = ctypes.c_size_t(), 4
    b = _Batch(P, P, P, 1, 4, ((1 << 31) - 1 - over) // heads, 1)
    c = cache(kv_heads=1)
    assert lib.nnq_kv_attention_workspace(ctx, ctypes.byref(c), ctypes.byref(b), heads, ctypes.byref(need)) == status


@pytest.mark.parametrize("kind,names", [(KvCache, ("k", "v", "k_exp", "v_exp")), (KvBatch, ("table", "length", "row_start", "slot", "position", "used", "rows"))])
def test_tensors_that_calls_rely_on_are_not_replaced(kind, names):
    """A cache's addresses go into every call, and a batch writes as many rows as its first slot map has."""
    for name in names:
        with pytest.raises(AttributeError):
            setattr(kind.__new__(kind), name, None)
