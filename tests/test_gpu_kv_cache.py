"""Block tables, append and read of the paged 8-bit cache, and attention over it, against the definitions in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nn_b200 import api, kv_cache
from tests import kv_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMATS = [kv_cache.INT8, kv_cache.E4M3]


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------
# tables
# ------------------------------------------------------------------------------------------


def plain_tables(past, count, free, skip, block, table, rows):
    """The step's tables, one request after another."""
    table, at, slot, position, start = table.copy(), skip, [], [], [0]
    for r, (p, c) in enumerate(zip(past, count)):
        c = max(c, 0)
        first = -(-p // block)
        for j in range(-(-(p + c) // block) - first):
            if first + j < table.shape[1]:
                table[r, first + j] = free[at] if at < len(free) else -1
            at += 1
        for t in range(p, p + c):
            b = table[r, t // block] if t // block < table.shape[1] else -1
            slot.append(b * block + t % block if b >= 0 else -1)
            position.append(t)
        start.append(start[-1] + c)
    slot, position = (slot + [-1] * rows)[:rows], (position + [-1] * rows)[:rows]
    return table, [p + max(c, 0) for p, c in zip(past, count)], start, slot, position, at


def check_tables(past, count, block, *, spare=2, skip=0, rows=None, width=None, free=None, alias=False):
    rng = np.random.default_rng(len(past) * 7 + block)
    need = [-(-(p + max(c, 0)) // block) for p, c in zip(past, count)]
    old = [-(-p // block) for p in past]
    width = max(need) + 1 if width is None else width
    order = rng.permutation(sum(need) + spare + skip + 5).astype(np.int32)
    table = np.full((len(past), width), -7, np.int32)
    at = 0
    for r, n in enumerate(old):
        table[r, :n] = order[at:at + n][:max(0, width)]
        at += n
    free = order[at:at + skip + sum(need) - sum(old) + spare] if free is None else np.asarray(free, np.int32)
    rows = sum(max(c, 0) for c in count) if rows is None else rows
    want = plain_tables(past, count, list(free), skip, block, table, rows)
    b = kv_cache.KvBatch(len(past), width, rows, block)
    b.table.copy_(i32(table))
    p, s = i32(past), i32([skip])
    if alias:
        b.length.copy_(p)
        b.used.copy_(s)
        p, s = b.length, b.used
    b.build(p, i32(count), i32(free), s)
    for name, w in zip(("table", "length", "row_start", "slot", "position", "used"), want):
        assert np.array_equal(getattr(b, name).cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name
    return b


@pytest.mark.parametrize("block", [16, 64, 256])
@pytest.mark.parametrize("requests", [1, 2, 31, 257, 2049, 5000])
def test_tables_of_a_decode_step(requests, block):
    rng = np.random.default_rng(requests)
    check_tables(rng.integers(0, 700, requests).tolist(), [1] * requests, block)


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("most,requests", [(3, 40), (900, 7), (4000, 30), (1, 3000)])
def test_tables_of_mixed_requests(most, requests, alias):
    rng = np.random.default_rng(most)
    check_tables(rng.integers(0, 500, requests).tolist(), rng.integers(-1, most + 1, requests).tolist(), 32, skip=3, alias=alias)


def test_tables_at_block_edges_and_without_tokens():
    past = [0, 0, 15, 16, 17, 31, 32, 0, 16]
    check_tables(past, [1, 16, 1, 1, 15, 2, 0, 17, 16], 16)
    check_tables(past, [0] * 9, 16)
    check_tables([0], [0], 16, rows=0)
    check_tables([5], [3], 16, rows=9)                    # rows behind the last request
    check_tables([5, 40], [30, 40], 16, rows=33)          # fewer rows than tokens


def test_tables_without_room():
    b = check_tables([3, 10, 0], [40, 30, 20], 16, free=[50, 51, 52])            # the list ends
    assert int(b.used) == 2 + 2 + 2 and (b.slot.cpu().numpy() == -1).any()
    check_tables([3, 10, 0], [40, 30, 20], 16, free=[])
    check_tables([3, 60], [100, 10], 16, width=4)                                # the table's row ends
    check_tables([2], [5], 256, free=[(1 << 31) // 256], skip=0)                  # (a slot beyond 31 bits would need the block used: it is not)
    b = check_tables([0], [1], 16, free=[7], skip=5)                             # everything taken
    assert int(b.used) == 6 and int(b.slot[0]) == -1


def test_a_block_number_whose_slots_pass_31_bits_gives_none():
    b = kv_cache.KvBatch(1, 2, 1, 256)
    b.build(i32([0]), i32([1]), i32([1 << 23]))
    assert int(b.slot[0]) == -1


def test_a_captured_step_advances_the_batch():
    block, n = 16, 5
    past = [14, 0, 31, 100, 15]
    order = np.random.default_rng(1).permutation(200).astype(np.int32)
    b = kv_cache.KvBatch(n, 20, n, block)
    want = np.full((n, 20), -1, np.int32)
    at = 0
    for r, p in enumerate(past):
        k = -(-p // block)
        want[r, :k] = order[at:at + k]
        at += k
    b.table.copy_(i32(want))
    b.length.copy_(i32(past))
    one, free = i32([1] * n), i32(order[at:])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            b.build(b.length, one, free, b.used)
        for _ in range(40):
            g.replay()
    torch.cuda.synchronize()
    used = 0
    for step in range(40):
        want, past, _, slot, _, used = plain_tables(past, [1] * n, order[at:].tolist(), used, block, want, n)
    assert np.array_equal(b.table.cpu().numpy(), want) and b.length.tolist() == past and b.slot.tolist() == slot and int(b.used) == used


def test_tables_refuse_wrong_tensors():
    b = kv_cache.KvBatch(3, 4, 3, 16)
    ok = i32([1, 1, 1])
    for args in ((ok.long(), ok, ok), (ok[:2], ok, ok), (ok, ok.cpu(), ok), (ok, ok, ok.float()), (ok, ok, ok, i32([1, 2]))):
        with pytest.raises(api.TensorError):
            b.build(*args)
    with pytest.raises(api.Unsupported):
        kv_cache.KvBatch(3, 4, 3, 48).build(ok, ok, ok)
    with pytest.raises(api.InvalidArgument):
        kv_cache.KvBatch.from_tensors(b.table, b.length, b.row_start, 16).build(ok, ok, ok)


# ------------------------------------------------------------------------------------------
# append and read
# ------------------------------------------------------------------------------------------


def filled_cache(rng, fmt, blocks, heads, dim, block):
    """A cache with a random byte everywhere (valid exponents), and its copy in numpy."""
    c = kv_cache.KvCache(blocks, heads, dim, block, fmt)
    for t in (c.k, c.v):
        t.copy_(torch.from_numpy(rng.integers(0, 256, t.shape, dtype=np.uint8)))
    for t in (c.k_exp, c.v_exp):
        t.copy_(torch.from_numpy(rng.integers(112, 125, t.shape).astype(np.uint8)))
    return c


def values_of(c):
    fmt = c.fmt
    return [ref.decode(fmt, t.cpu().numpy(), e.cpu().numpy()) for t, e in ((c.k, c.k_exp), (c.v, c.v_exp))]


def check_append(c, k, v, slots):
    """Appends and compares the whole cache, bytes that no row concerns included."""
    before = [t.cpu().numpy().copy() for t in (c.k, c.v)]
    want, exps = values_of(c), [e.cpu().numpy().copy() for e in (c.k_exp, c.v_exp)]
    for i, x in enumerate((k, v)):
        ref.append(c.fmt, want[i], exps[i], x.float().cpu().numpy(), list(slots), c.block)
    c.append(k, v, i32(slots))
    got = values_of(c)
    touched = np.zeros(c.blocks, bool)
    touched[[s // c.block for s in slots if s >= 0]] = True
    for i in range(2):
        assert np.array_equal((c.k_exp, c.v_exp)[i].cpu().numpy(), exps[i])
        assert np.array_equal(got[i], want[i])
        assert np.array_equal((c.k, c.v)[i].cpu().numpy()[~touched], before[i][~touched])
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,block", [(64, 1, 16), (128, 8, 16), (128, 2, 256), (192, 3, 64), (256, 2, 32)])
def test_append_of_single_tokens_grows_the_scales(fmt, dtype, dim, heads, block):
    rng = np.random.default_rng(dim + block)
    c = filled_cache(rng, fmt, 12, heads, dim, block)
    for step in range(3):
        blocks = rng.permutation(12)[:9]
        slots = [int(b * block + rng.integers(0, block)) for b in blocks]
        slots[2], slots[5] = blocks[2] * block, blocks[5] * block + block - 1
        slots[7] = -1
        size = np.exp(rng.normal(0, 3, (9, heads, 1)))
        k, v = (torch.from_numpy((rng.standard_normal((9, heads, dim)) * size).astype(np.float32)).to(DEV, dtype) for _ in range(2))
        check_append(c, k, v, slots)
    c.backend.device_status()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("block", [16, 64, 256])
@pytest.mark.parametrize("rows", [1, 7, 8, 9, 40, 300, 700])
def test_append_of_prompts(fmt, block, rows):
    """Two requests' rows one after the other, the first behind tokens that its first block holds."""
    rng = np.random.default_rng(rows + block)
    heads, dim = 2, 64
    table = rng.permutation(100)
    c = filled_cache(rng, fmt, 100, heads, dim, block)
    first, slots, at = rows * 2 // 3, [], 0
    for start, n in ((5, first), (0, rows - first)):
        p = np.arange(start, start + n)
        slots += [int(table[at + x // block] * block + x % block) for x in p]
        at += (start + n) // block + 1
    k, v = (torch.from_numpy((rng.standard_normal((rows, heads, dim)) * 2).astype(np.float32)).to(DEV) for _ in range(2))
    check_append(c, k, v, slots)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_at_the_edges_of_the_numbers(fmt):
    """Largest values on a scale's border, zeros, numbers near both ends of f32, ties."""
    heads, dim = 1, 64
    rng = np.random.default_rng(5)
    c = filled_cache(rng, fmt, 40, heads, dim, 16)
    top = ref.TOP[fmt]
    rows = []
    for big in (0.0, 1.0, top, np.nextafter(np.float32(top), np.float32(1e9)), top / 2, 2.0, 1.984375, 1.75, 3.4e38, 1e38, 1e-38, 1e-45, 2.0 ** -120 * top):
        x = rng.uniform(-1, 1, dim).astype(np.float32) * np.float32(big)
        x[3] = -big
        with np.errstate(over="ignore"):   # (3.4e38 and 1e38: to infinity)
            x[4:20] = np.float32(big) * (np.arange(16) + 0.5).astype(np.float32) / 128
        rows.append(x)
    x = torch.from_numpy(np.stack(rows).astype(np.float32)[:, None]).to(DEV)
    check_append(c, x, x.flip(0).contiguous(), [16 * i + (i % 3) * 5 for i in range(len(rows))])
    with pytest.raises(api.ValueOutOfRange):
        c.backend.device_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_values_that_are_not_finite_are_stored_and_reported(fmt):
    rng = np.random.default_rng(6)
    c = filled_cache(rng, fmt, 4, 2, 64, 16)
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    x[0, 0, 5], x[1, 1, 6], x[1, 1, 7], x[2, 0] = np.nan, np.inf, -np.inf, np.nan
    k = torch.from_numpy(x).to(DEV)
    check_append(c, k, torch.ones_like(k), [3, 16, 40])
    with pytest.raises(api.ValueOutOfRange):
        c.backend.device_status()
    c.backend.device_status()


def test_slots_beyond_the_cache_are_skipped_and_reported():
    c = filled_cache(np.random.default_rng(7), 0, 4, 1, 64, 16)
    x = torch.randn(3, 1, 64, device=DEV)
    before = c.k.clone(), c.k_exp.clone()
    c.append(x, x, i32([64, 2 ** 31 - 1, 65]))
    with pytest.raises(api.InvalidArgument):
        c.backend.device_status()
    assert torch.equal(c.k, before[0]) and torch.equal(c.k_exp, before[1])
    k, v = c.read(i32([64, -1, 5]))
    with pytest.raises(api.InvalidArgument):
        c.backend.device_status()
    assert not k[:2].any() and not v[:2].any() and k[2].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_read_gives_every_code_exactly(fmt, dtype):
    rng = np.random.default_rng(8)
    c = filled_cache(rng, fmt, 6, 3, 192, 32)
    c.k.view(-1)[:256] = torch.arange(256, dtype=torch.uint8, device=DEV)
    slots = rng.permutation(6 * 32).tolist() + [-1, 0, 0]
    k, v = c.read(i32(slots), dtype)
    for got, want in zip((k, v), values_of(c)):
        for i, s in enumerate(slots):
            w = want[s // 32, :, s % 32] if s >= 0 else np.zeros((3, 192))
            assert np.array_equal(got[i].double().cpu().numpy(), w)


def test_rows_of_a_wider_product_and_other_layouts():
    """k and v as slices of one [rows, (heads + 2 kv) dim] tensor, transposed heads, an odd offset, other dtypes."""
    rng = np.random.default_rng(9)
    c = filled_cache(rng, 0, 8, 2, 64, 16)
    qkv = torch.randn(5, 8, 64, device=DEV)
    check_append(c, qkv[:, 4:6], qkv[:, 6:8], [3, 4, 5, 33, 34])
    x = torch.randn(2, 5, 64, device=DEV).transpose(0, 1)
    check_append(c, x, x, [7, 8, 50, 51, 52])
    odd = torch.randn(5 * 128 + 1, device=DEV)[1:].view(5, 2, 64)
    check_append(c, odd, odd.bfloat16(), [9, 10, 11, 12, 13])
    half = odd.half()
    check_append(c, half, half, [64, 65, 66, 67, 68])
    one = odd[:1].expand(5, 2, 64)   # rows of stride 0
    check_append(c, one, one, [80, 81, 82, 83, 84])


def test_append_and_read_refuse_wrong_tensors():
    c = kv_cache.KvCache(4, 2, 64)
    x, s = torch.zeros(3, 2, 64, device=DEV), i32([0, 1, 2])
    for args in ((x[:, :1], x, s), (x, x[:2], s), (x, x, s[:2]), (x, x, s.long()), (x.cpu(), x, s), (x.view(3, 128), x, s)):
        with pytest.raises(api.TensorError):
            c.append(*args)
    with pytest.raises(api.TensorError):
        c.read(s, torch.float16)
    for kw in (dict(dim=96), dict(block=20), dict(fmt=3), dict(blocks=0), dict(blocks=1 << 28)):
        with pytest.raises(api.TensorError):
            kv_cache.KvCache(**{**dict(blocks=2, kv_heads=1, dim=64), **kw})


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------


def serving(rng, fmt, lengths, rows, *, heads, kv, dim, block, dtype=torch.float32, spare=0, scale_spread=3):
    """A cache whose blocks lie in any order among others full of arbitrary bytes, tables, and queries of `rows` rows per request."""
    need = [-(-n // block) for n in lengths]
    order = rng.permutation(sum(need) + 4)
    c = filled_cache(rng, fmt, sum(need) + 4, kv, dim, block)
    for e in (c.k_exp, c.v_exp):   # values of about one
        e.copy_(torch.from_numpy(rng.integers(121 - scale_spread, 122, e.shape).astype(np.uint8)))
    table, at = np.full((len(lengths), max(max(need), 1)), -1, np.int32), 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((int(start[-1]) + spare, heads, dim)).astype(np.float32)).to(DEV, dtype)
    return c, table, start, q, kv_cache.KvBatch.from_tensors(i32(table), i32(lengths), i32(start), block)


def bound(mag, want, top, dim, length, out_dtype, largest, one_term):
    """How far an output may be off, element by element (mag = sum p |v|).

    Scores: products are exact or carry two f16 terms (2^-21 of |q||k| for f32 queries), sums of dim / 16 steps round by 2^-23 of the
    magnitude each, the scalings and the difference to the reference by 2^-23 of it in all: delta = top (2^-20 + dim / 16 * 2^-23), top
    the largest sum |q||k| * scale. A weight is then off by 2 delta relative (numerator and normalisation), its exponential by 2^-21, its
    two f16 terms by 2^-22; the sums of a warp's steps round by 2^-23 each. Joining warps and parts: 2^-20. A factor of two on all.

    Below that a weight has a floor: its second f16 term is a multiple of 2^-24, so it is off by up to 2^-25 where the largest of the
    row is 1 or more and their sum too. `length` keys of values up to `largest` make that length * 2^-25 * largest, which counts for
    dimensions in which the heavy keys are zero.

    bf16 queries and outputs in numbers that make a prompt: a weight is one f16 number, off by half a step, 2^-11 of itself: 2^-11 mag."""
    eps = 2 * (top * (2.0 ** -20 + dim / 16 * 2.0 ** -23)) + 2.0 ** -19 + (length / 16 + 64) * 2.0 ** -23
    half_step = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24
    if one_term:
        eps += 2.0 ** -12
    return 2 * eps * mag + half_step * np.abs(want) + length * 2.0 ** -25 * largest


def check_attend(c, table, lengths, start, q, batch, *, scale=None, window=0, max_rows=None, out=None):
    n = int(start[-1])
    max_rows = int(np.max(np.diff(start))) if max_rows is None else max_rows
    k, v = values_of(c)
    y = c.attend(q, batch, scale, window, max_rows, out)
    want, mag, top = ref.attend(q.double().cpu().numpy()[:n], k, v, table, lengths, start, c.block, c.dim ** -0.5 if scale is None else scale, window)
    got = y.double().cpu().numpy()[:n]
    lim = bound(mag, want, top, c.dim, max(lengths), y.dtype, np.abs(v).max(), q.dtype == y.dtype == torch.bfloat16 and max_rows * q.shape[1] // c.kv_heads > 32)
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], lim[bad][:4])
    c.backend.device_status()
    return y


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 3, 4, 8, 11])
def test_attention_of_single_tokens(fmt, dtype, dim, group):
    rng = np.random.default_rng(dim + group)
    lengths = [1, 15, 16, 17, 130, 63, 300]
    c, table, start, q, b = serving(rng, fmt, lengths, [1] * 7, heads=2 * group, kv=2, dim=dim, block=16, dtype=dtype)
    check_attend(c, table, lengths, start, q, b)


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 100])
def test_attention_of_a_few_rows(block, window):
    """Rows of different requests in different numbers, some with none, lengths that end inside a block, windows that begin in one."""
    rng = np.random.default_rng(block + window)
    lengths, rows = [40, 7, 300, 128, 5, 257], [5, 7, 2, 0, 1, 9]
    c, table, start, q, b = serving(rng, block % 3 % 2, lengths, rows, heads=6, kv=2, dim=64, block=block)
    check_attend(c, table, lengths, start, q, b, window=window)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("group,dim,dtype", [(1, 64, torch.float32), (4, 128, torch.bfloat16), (4, 128, torch.float32), (7, 128, torch.bfloat16), (2, 192, torch.bfloat16), (3, 256, torch.float32)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_of_prompts(fmt, group, dim, dtype, window):
    rng = np.random.default_rng(group + dim)
    lengths, rows = [150, 33, 90], [150, 1, 70]
    c, table, start, q, b = serving(rng, fmt, lengths, rows, heads=2 * group, kv=2, dim=dim, block=32, dtype=dtype)
    check_attend(c, table, lengths, start, q, b, window=window)


@pytest.mark.parametrize("group,dim,rows", [(71, 64, 1), (128, 128, 1), (65, 192, 1), (33, 128, 2), (16, 64, 4), (13, 64, 5)])
def test_attention_of_many_heads_to_one(group, dim, rows):
    """Up to 64 query vectors of a request and key / value head, and more: single tokens of many heads among them."""
    rng = np.random.default_rng(group)
    lengths = [100, 7, 33]
    c, table, start, q, b = serving(rng, 1, lengths, [rows, 1, rows], heads=group, kv=1, dim=dim, block=32, dtype=torch.bfloat16)
    check_attend(c, table, lengths, start, q, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,window", [(5, 0), (8, 0), (5, 2044)])
def test_attention_of_a_few_rows_of_long_requests(rows, window, dtype):
    """33 to 64 query vectors: requests of 2^16 keys (times heads and requests) and more take another kernel than shorter ones do."""
    rng = np.random.default_rng(rows)
    lengths = [2100, 2047, 2048, 5]
    c, table, start, q, b = serving(rng, 1, lengths, [rows, rows, rows, 5], heads=64, kv=8, dim=64, block=64, dtype=dtype)
    check_attend(c, table, lengths, start, q, b, window=window)


@pytest.mark.parametrize("window", [1, 2 ** 31 - 1])
def test_attention_of_rows_before_the_first_position(window):
    """A request of more rows than positions: the rows before position 0 see nothing, whatever the window is."""
    rng = np.random.default_rng(3)
    lengths = [90, 100]
    c, table, start, q, b = serving(rng, 1, lengths, [90, 100], heads=8, kv=2, dim=64, block=32, dtype=torch.float32)
    check_attend(c, table, lengths, start, q, b, window=window)
    b.length[0] = 20
    check_attend(c, table, [20, 100], start, q, b, window=window)


@pytest.mark.parametrize("count,length", [(1, 6001), (3, 2500), (200, 40)])
def test_attention_that_is_cut_into_parts(count, length):
    """Long requests in many parts, and many short ones in one."""
    rng = np.random.default_rng(count)
    lengths = [length - 7 * i % length for i in range(count)]
    c, table, start, q, b = serving(rng, 0, lengths, [1] * count, heads=4, kv=1, dim=128, block=64)
    y = check_attend(c, table, lengths, start, q, b)
    for _ in range(3):   # the same bits every time
        assert torch.equal(y, c.attend(q, b))


def test_requests_of_no_tokens_and_rows_of_none():
    rng = np.random.default_rng(3)
    lengths, rows = [0, 2, 20, 0], [2, 4, 1, 0]   # rows that stand before position 0 see nothing
    c, table, start, q, b = serving(rng, 1, lengths, rows, heads=4, kv=2, dim=64, block=16, spare=3)
    out = torch.full((10, 4, 64), 7.0, device=DEV)
    y = check_attend(c, table, lengths, start, q, b, out=out)
    assert y is out and not y[:4].any() and (y[7:] == 7.0).all()


def test_more_requests_than_a_block_has_threads():
    rng = np.random.default_rng(4)
    lengths = rng.integers(1, 60, 700).tolist()
    c, table, start, q, b = serving(rng, 0, lengths, [1] * 700, heads=2, kv=2, dim=64, block=16)
    check_attend(c, table, lengths, start, q, b)


@pytest.mark.parametrize("rows", [1, 40])
def test_scales_far_apart(rows):
    """Blocks whose exponents differ by up to 2^60, so that most weigh nothing and few carry the result."""
    rng = np.random.default_rng(11)
    lengths = [200]
    c, table, start, q, b = serving(rng, 0, lengths, [rows], heads=4, kv=2, dim=64, block=16)
    c.v_exp.copy_(torch.from_numpy(rng.integers(90, 150, c.v_exp.shape).astype(np.uint8)))
    check_attend(c, table, lengths, start, q, b)
    c.v_exp.fill_(1)   # the smallest numbers
    check_attend(c, table, lengths, start, q, b)


@pytest.mark.parametrize("rows", [1, 40])
def test_sharp_and_flat_softmax(rows):
    rng = np.random.default_rng(12)
    lengths = [500]
    c, table, start, q, b = serving(rng, 0, lengths, [rows], heads=4, kv=2, dim=64, block=32)
    check_attend(c, table, lengths, start, q * 60, b)
    check_attend(c, table, lengths, start, q * 1e-20, b)
    check_attend(c, table, lengths, start, q * 0, b)
    check_attend(c, table, lengths, start, q, b, scale=3.0)


@pytest.mark.parametrize("rows", [1, 3, 50])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_concerns_its_own_head_alone(rows, what):
    rng = np.random.default_rng(13)
    lengths = [90, 60]
    c, table, start, q, b = serving(rng, 1, lengths, [rows, rows], heads=4, kv=2, dim=64, block=16)
    clean = c.attend(q, b, max_rows=rows)
    q2 = q.clone()
    q2[rows - 1, 1, 3] = what
    got = c.attend(q2, b, max_rows=rows)
    assert got[rows - 1, 1].isnan().all()
    got[rows - 1, 1] = clean[rows - 1, 1]
    # (its scores may move the references of a warp's other vectors: both results are within `bound`, 2^-16 of the largest value)
    assert float((got - clean).abs().max()) <= 2 * 2.0 ** -16 * float(np.abs(values_of(c)[1]).max())


@pytest.mark.parametrize("rows", [1, 40])
def test_blocks_that_do_not_exist_count_as_unseen(rows):
    rng = np.random.default_rng(14)
    lengths = [100, 80]
    c, table, start, q, b = serving(rng, 0, lengths, [rows, rows], heads=2, kv=1, dim=64, block=16)
    table[0, 2], table[0, 4], table[1, 0] = -1, c.blocks, 2 ** 31 - 1
    b.table.copy_(i32(table))
    with pytest.raises(api.InvalidArgument):
        check_attend(c, table, lengths, start, q, b)
    table[:] = -1
    b.table.copy_(i32(table))
    assert not c.attend(q, b, max_rows=rows).any()
    with pytest.raises(api.InvalidArgument):
        c.backend.device_status()


@pytest.mark.parametrize("rows", [1, 40])
def test_numbers_of_a_batch_outside_its_tensors_do_no_harm(rows):
    """Lengths beyond the table, row numbers beyond the rows, descending ones: reported, and nothing else is touched."""
    rng = np.random.default_rng(15)
    lengths = [60, 50]
    c, table, start, q, b = serving(rng, 0, lengths, [rows, rows], heads=2, kv=1, dim=64, block=16)
    for length, row in (([10 ** 6, 50], start), ([60, -5], start), ([60, 50], [0, rows, 10 ** 6]), ([60, 50], [rows, 0, 2 * rows]), ([60, 50], [-3, rows, rows])):
        b.length.copy_(i32(length))
        b.row_start.copy_(i32(row))
        wide = torch.full((2 * rows + 8, 2, 64), 3.0, device=DEV)
        c.attend(q, b, max_rows=rows, out=wide[:2 * rows])
        assert (wide[2 * rows:] == 3.0).all()
        if length[1] != -5:
            with pytest.raises(api.InvalidArgument):
                c.backend.device_status()
        else:
            try:
                c.backend.device_status()
            except api.InvalidArgument:
                pass


@pytest.mark.parametrize("rows", [1, 60])
def test_max_rows_chooses_kernels_not_results(rows):
    rng = np.random.default_rng(16)
    lengths = [200, 70]
    c, table, start, q, b = serving(rng, 0, lengths, [rows, 1], heads=8, kv=2, dim=128, block=16)
    for m in (1, 2, rows, 1000):
        check_attend(c, table, lengths, start, q, b, max_rows=m)


def test_rows_of_queries_in_a_wider_tensor_and_outputs_in_another():
    rng = np.random.default_rng(17)
    lengths = [70, 30]
    c, table, start, q, b = serving(rng, 0, lengths, [1, 2], heads=4, kv=2, dim=64, block=16)
    qkv = torch.cat([q, torch.randn(3, 4, 64, device=DEV)], 1)
    out = torch.zeros(3, 6, 64, device=DEV, dtype=torch.bfloat16)
    y = check_attend(c, table, lengths, start, qkv[:, :4], b, out=out[:, 1:5])
    assert y.dtype == torch.bfloat16 and not out[:, 0].any() and not out[:, 5].any()
    check_attend(c, table, lengths, start, q.transpose(0, 1).contiguous().transpose(0, 1), b)


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_on_another_stream_and_in_two_graphs(rows):
    """Two captured calls of different inputs replayed together: neither sees the other's records."""
    rng = np.random.default_rng(18)
    lengths = [3000]
    c, table, start, q, b = serving(rng, 0, lengths, [rows], heads=4, kv=2, dim=64, block=16)
    q2 = q * 0.5 + 1
    want = c.attend(q, b, max_rows=rows).clone(), c.attend(q2, b, max_rows=rows).clone()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for s, x in zip(streams, (q, q2)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(c.attend(x, b, max_rows=rows))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_step_captured_whole():
    """Tables that advance, append and attention in one graph: twenty tokens of two requests against one call with all of them."""
    rng = np.random.default_rng(21)
    block, n = 16, 2
    c = kv_cache.KvCache(12, 2, 64, block)
    b = kv_cache.KvBatch(n, 6, n, block)
    k, v, q = (torch.from_numpy(rng.standard_normal((20, n, h, 64)).astype(np.float32)).to(DEV) for h in (2, 2, 4))
    now = [torch.zeros_like(x[0]) for x in (k, v, q)]
    one, free = i32([1, 1]), i32(rng.permutation(12))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            b.build(b.length, one, free, b.used)
            c.append(now[0], now[1], b.slot)
            y = c.attend(now[2], b)
        outs = []
        for t in range(20):
            for dst, src in zip(now, (k, v, q)):
                dst.copy_(src[t])
            g.replay()
            outs.append(y.clone())
    torch.cuda.synchronize()
    assert b.length.tolist() == [20, 20] and int(b.used) == 4
    kk, vv = values_of(c)
    want, mag, top = ref.attend(now[2].double().cpu().numpy(), kk, vv, b.table.cpu().numpy(), [20, 20], [0, 1, 2], block, 0.125, 0)
    got = outs[-1].double().cpu().numpy()
    assert (np.abs(got - want) <= bound(mag, want, top, 64, 20, torch.float32, np.abs(vv).max(), False)).all()
    c.backend.device_status()


def test_attention_refuses_wrong_tensors():
    c = kv_cache.KvCache(4, 2, 64)
    b = kv_cache.KvBatch(1, 4, 1, 16)
    q = torch.zeros(1, 4, 64, device=DEV)
    for args, kw in (((q[:, :3], b), {}), ((q[:, :, :32], b), {}), ((q[0], b), {}), ((q.cpu(), b), {}), ((q, b), dict(window=-1)), ((q, b), dict(scale=0.0)),
                     ((q, kv_cache.KvBatch(1, 4, 1, 32)), {}), ((q, b), dict(out=torch.zeros(2, 4, 64, device=DEV))),
                     ((q, b), dict(out=torch.zeros(1, 4, 64, device=DEV, dtype=torch.float16)))):
        with pytest.raises(api.TensorError):
            c.attend(*args, **kw)


@pytest.mark.parametrize("rows", [1, 40, 150])
@pytest.mark.parametrize("window,block", [(20, 16), (70, 16), (100, 16), (20, 32), (70, 32), (100, 64)])
def test_blocks_behind_every_window_may_have_been_given_back(rows, window, block):
    """Entries of blocks that no row of a request sees any more are -1: nothing reads them, and nothing is reported."""
    rng = np.random.default_rng(rows + window)
    lengths = [333, 150, 201]
    c, table, start, q, b = serving(rng, 1, lengths, [rows] * 3, heads=8, kv=2, dim=64, block=block)
    for r, n in enumerate(lengths):
        table[r, :max(0, n - rows - window + 1) // block] = -1
    assert (table[0, :1] == -1).all() and window > 1
    b.table.copy_(i32(table))
    check_attend(c, table, lengths, start, q, b, window=window)


@pytest.mark.parametrize("rows", [3, 90])
def test_caches_beyond_32_bits_of_bytes(rows):
    """The last blocks of a cache of 5 GB of codes, against a small cache with the same tokens."""
    kv, dim, block, need = 2, 128, 64, 2
    large, small = kv_cache.KvCache(320000, kv, dim, block), kv_cache.KvCache(need, kv, dim, block)
    assert large.k.numel() > 1 << 32
    k, v, q = torch.randn(rows, kv, dim, device=DEV), torch.randn(rows, kv, dim, device=DEV), torch.randn(rows, 8, dim, device=DEV)
    out = []
    for c, first in ((large, large.blocks - need), (small, 0)):
        slots = first * block + torch.arange(rows, dtype=torch.int32, device=DEV)
        c.append(k, v, slots)
        b = kv_cache.KvBatch.from_tensors(i32([[first, first + 1]]), i32([rows]), i32([0, rows]), block)
        out.append((*c.read(slots), c.attend(q, b, max_rows=rows)))
    assert all(torch.equal(x, y) for x, y in zip(*out)) and out[0][2].any()
    assert torch.equal(large.k[-need:], small.k) and torch.equal(large.v_exp[-need:], small.v_exp) and not large.k[:-need].any() and not large.v[:-need].any()
    large.backend.device_status()


@pytest.mark.parametrize("dtype,want", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float64, torch.float32)])
def test_types_of_queries_and_outputs(dtype, want):
    rng = np.random.default_rng(22)
    c, table, start, q, b = serving(rng, 0, [40, 30], [1, 1], heads=4, kv=2, dim=64, block=16)
    y = check_attend(c, table, [40, 30], start, q.to(dtype), b)
    assert y.dtype == want
    check_attend(c, table, [40, 30], start, q.to(dtype), b, out=torch.empty(2, 4, 64, dtype=torch.bfloat16, device=DEV))


@pytest.mark.parametrize("window", [-1, 2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_windows_beyond_31_bits_are_refused(window):
    c, b = kv_cache.KvCache(4, 2, 64), kv_cache.KvBatch(1, 4, 1, 16)
    with pytest.raises(api.InvalidArgument):
        c.attend(torch.zeros(1, 4, 64, device=DEV), b, window=window)


# ------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_batch_served_from_prompts_to_tokens(fmt):
    """Three requests: prompts, then ten steps of one token each with one request leaving and another joining; tables, append, attention
    and log probabilities as a server calls them, against f64 attention over the values that the cache holds."""
    from nn_b200 import logprobs
    rng = np.random.default_rng(20)
    block, kv, group, dim, blocks, vocab = 16, 2, 4, 64, 40, 1000
    c = kv_cache.KvCache(blocks, kv, dim, block, fmt)
    head = torch.randn(kv * group * dim, vocab, device=DEV) * 0.2
    free = rng.permutation(blocks).astype(np.int32)
    held, tables, taken = [0, 0, 0], np.full((3, 12), -1, np.int32), 0
    for step in range(12):
        count = [37, 5, 90] if step == 0 else [1, 1, 1] if step != 6 else [1, 0, 20]
        if step == 6:
            held[2] = 0   # the third request leaves (its blocks are not used again here) and a prompt takes its place
        rows = sum(count)
        b = kv_cache.KvBatch(3, 12, rows + 2, block)
        b.table.copy_(i32(tables))
        b.build(i32(held), i32(count), i32(free), i32([taken]))
        k, v = torch.randn(rows + 2, kv, dim, device=DEV), torch.randn(rows + 2, kv, dim, device=DEV)
        q = torch.randn(rows + 2, kv * group, dim, device=DEV)
        c.append(k, v, b.slot)
        tables, taken = b.table.cpu().numpy(), int(b.used)
        held = [h + n for h, n in zip(held, count)]
        start = np.concatenate([[0], np.cumsum(count)])
        y = check_attend(c, tables, held, start, q, b)
        # what was appended is what is attended to: half a step of a code is 2^-7 (int8) or 2^-4 (e4m3) of its block's largest
        kk, vv = c.read(b.slot[:rows])
        for got, x in ((kk, k[:rows]), (vv, v[:rows])):
            assert float((got - x).abs().max()) <= (2.0 ** -7 if fmt == 0 else 2.0 ** -4) * 6 * (1 if step == 0 else 3)
        last = torch.from_numpy(start[1:][np.diff(start) > 0] - 1).to(DEV)
        logits = y[last].flatten(1) @ head
        got = logprobs.token_logprobs(logits, logits.argmax(1), 3)
        lp, _, tt, _ = ref.logprobs(logits.cpu().numpy(), logits.argmax(1).cpu().numpy(), 3)
        assert np.abs(got.logprob.cpu().numpy() - lp).max() <= 1e-5 and np.array_equal(got.top_tokens.cpu().numpy(), tt)
    c.backend.device_status()
