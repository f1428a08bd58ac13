"""How many digits attention over the 8-bit cache keeps where they are easily lost: keys that weigh little beside one that weighs nearly all."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nn_b200 import kv_cache
from tests import kv_reference as ref
from tests.test_gpu_kv_cache import DEV, FORMATS, i32, serving, values_of

pytestmark = pytest.mark.gpu


def bound(mag, want, top, dim, keys, out_dtype, largest):
    """How far an output may be off, element by element: mag = sum p |v|, top the largest scale sum |q||k| of a vector, keys those that it sees.

    A score: products exact or of two f16 terms (2^-21), dim / 16 sums of 2^-23 each, scaling and reference 2^-23: delta = top (2^-20 +
    dim / 16 2^-23), which counts twice (weight and normalisation); exponentials 2^-21, weights of two terms 2^-22, the joining of warps and
    parts 2^-20: 2^-19 in all; the sums over keys 2^-23 for every 16 of them. A factor of two on all. A weight of two terms ends at a multiple of
    2^-24 under a reference that gives the largest 2^7 or more: off by 2^-25 at most, 2^-32 of the largest. Outputs are rounded once."""
    eps = 2 * top * (2.0 ** -20 + dim / 16 * 2.0 ** -23) + 2.0 ** -19 + keys / 16 * 2.0 ** -23
    half_step = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24
    return 2 * eps * mag + half_step * np.abs(want) + keys * 2.0 ** -32 * largest


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,requests", [(1, 64), (40, 16)])
@pytest.mark.parametrize("nats", [8.0, 16.0, 17.5, 20.0])
def test_keys_under_a_sink(fmt, dtype, rows, requests, nats):
    """The first key of every request is `nats` above the others and its value is zero, as models come to use the first token of a context:
    what is attended to in earnest has weights of e^-nats, and all of the output is theirs."""
    rng = np.random.default_rng(int(nats * 2) + rows)
    lengths, heads, dim, block = [1100] * requests, 4, 64, 16
    c, table, start, q, b = serving(rng, fmt, lengths, [rows] * requests, heads=heads, kv=heads, dim=dim, block=block, dtype=dtype)
    one = 1.0 if fmt == kv_cache.INT8 else 4.0   # (values of 64 to 127 for int8, 256 to 448 for e4m3)
    kinds = np.arange(256)[(ref.VALUES[fmt] >= 64 * one) & (ref.VALUES[fmt] <= ref.TOP[fmt])].astype(np.uint8)
    small = np.arange(256)[np.abs(ref.VALUES[fmt]) <= 16 * one].astype(np.uint8)
    k, v = rng.choice(small, c.k.shape), rng.choice(kinds, c.v.shape)
    k[..., 0] = 0
    first = table[:, 0]
    k[first, :, 0] = 0
    k[first, :, 0, 0] = np.argmax(np.where(ref.VALUES[fmt] <= ref.TOP[fmt], ref.VALUES[fmt], 0))
    v[first, :, 0] = 0
    c.k.copy_(torch.from_numpy(k))
    c.v.copy_(torch.from_numpy(v))
    for e in (c.k_exp, c.v_exp):
        e.fill_(121 if fmt == kv_cache.INT8 else 119)   # values up to about two
    q[:, :, 0] = nats * dim ** 0.5 / float(ref.TOP[fmt] * 2.0 ** (-6 if fmt == kv_cache.INT8 else -8))
    y = c.attend(q, b, max_rows=rows)
    want, mag, top = ref.attend(q.double().cpu().numpy(), *values_of(c), table, lengths, start, block, dim ** -0.5, 0)
    lim = bound(mag, want, top, dim, 1100, dtype, 2.0)
    off = np.abs(y.double().cpu().numpy() - want)
    print(f"largest error {off.max() / np.abs(want).max():.2e} of the largest output")
    assert (off <= lim).all(), (off.max(), (off / lim).max())
    c.backend.device_status()


def exact(c, table, q, length, rows):
    """A single request's outputs and sum p |v| in 64 bits, on the device."""
    values = torch.from_numpy(ref.VALUES[c.fmt]).to(DEV)
    p = torch.arange(length, device=DEV)
    blk, off, e = i32(table[0]).long()[p // c.block], p % c.block, torch.arange(-127, 129, device=DEV).double()
    k, v = (values[t[blk, :, off].long()] * torch.exp2(e)[x[blk].long()][:, :, None] for t, x in ((c.k, c.k_exp), (c.v, c.v_exp)))   # [length, kv, dim]
    group = q.shape[1] // c.kv_heads
    y, mag = torch.empty(q.shape, dtype=torch.float64, device=DEV), torch.empty(q.shape, dtype=torch.float64, device=DEV)
    unseen = p[None] > torch.arange(length - rows, length, device=DEV)[:, None]
    for h in range(q.shape[1]):
        s = (q[:, h].double() @ k[:, h // group].T * c.dim ** -0.5).masked_fill_(unseen, -float("inf"))
        w = torch.softmax(s, 1)
        y[:, h], mag[:, h] = w @ v[:, h // group], w @ v[:, h // group].abs()
    return y, mag


@pytest.mark.parametrize("fmt,dim", [(kv_cache.INT8, 64), (kv_cache.E4M3, 128)])
@pytest.mark.parametrize("rows", [1, 72])
@pytest.mark.parametrize("length", [3000, 12001, 32000])
def test_sums_in_f32_do_not_lean_with_the_length(fmt, dim, rows, length):
    """Values of one sign, 32 heads (so that a part of the work is hundreds of keys): whatever the tensor core cuts off its sums shows in
    the mean error. A product added to a sum loses half a unit of 2^-23 of it on average, the sum grows from nothing, and at most 64 are added
    (two terms of a weight, 16 keys each): 64 * 2^-24 / 2 = 1.9e-6. Other roundings are as often up as down."""
    rng = np.random.default_rng(length + rows)
    c, table, start, q, b = serving(rng, fmt, [length], [rows], heads=32, kv=32, dim=dim, block=64)
    c.v.bitwise_and_(0x7F)   # positive codes (e4m3's 0x7F reads as 480)
    y = c.attend(q, b, max_rows=rows).double()
    want, mag = exact(c, table, q, length, rows)
    off = (y - want) / mag
    print(f"mean {float(off.mean()):.2e}, root mean square {float(off.square().mean().sqrt()):.2e}, largest {float(off.abs().max()):.2e}")
    assert abs(float(off.mean())) <= 2e-6
    assert float(off.square().mean().sqrt()) <= 2.5e-6   # (the lean and what is left of some hundred roundings of 2^-23)
    c.backend.device_status()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,dim", [(1, 64), (40, 64), (40, 128), (150, 128)])
@pytest.mark.parametrize("window", [2, 5, 40])
def test_outputs_in_bf16_are_the_exact_ones_rounded(fmt, rows, dim, window):
    """Whatever a request's rows are: no rounding to fewer bits stands in front of the one to bf16. Few keys, so that none averages away."""
    rng = np.random.default_rng(window + rows)
    lengths = [300, 200]
    c, table, start, q, b = serving(rng, fmt, lengths, [rows, rows], heads=8, kv=2, dim=dim, block=32, dtype=torch.bfloat16)
    y = c.attend(q, b, window=window, max_rows=rows).cpu()
    k, v = values_of(c)
    want, mag, top = ref.attend(q.double().cpu().numpy(), k, v, table, lengths, start, 32, dim ** -0.5, window)
    lim = bound(mag, want, top, dim, window, torch.float32, np.abs(v).max())
    low, high = (torch.from_numpy(x).to(torch.bfloat16) for x in (want - lim, want + lim))
    wrong = ~((low <= y) & (y <= high))
    assert not wrong.any(), (int(wrong.sum()), wrong.numel())
    c.backend.device_status()


@pytest.mark.parametrize("fmt,dim", [(kv_cache.INT8, 64), (kv_cache.E4M3, 128)])
@pytest.mark.parametrize("window", [0, 20, 300])
def test_chains_in_which_some_rows_see_nothing(fmt, dim, window):
    """f32 prompts whose sums leave tensor memory on the way: rows that see their first key behind that, blocks whose scales are far apart, so that
    the references move by much between two chains, rows in front of position 0, and a query that is not finite."""
    rng = np.random.default_rng(window + dim)
    lengths, rows = [700, 200], [300, 260]
    c, table, start, q, b = serving(rng, fmt, lengths, rows, heads=2, kv=2, dim=dim, block=32)
    for _ in range(2):
        y = c.attend(q, b, window=window, max_rows=300)
        want, mag, top = ref.attend(q.double().cpu().numpy(), *values_of(c), table, lengths, start, 32, dim ** -0.5, window)
        lim = bound(mag, want, top, dim, min(window or 700, 700), torch.float32, np.abs(values_of(c)[1]).max())
        off = np.abs(y.double().cpu().numpy() - want)
        assert (off <= lim).all(), float((off / lim).max())
        assert not y[300:360].any()
        q2 = q.clone()
        q2[280, 1, 3], q2[290, 0, 7] = float("nan"), float("inf")
        got = c.attend(q2, b, window=window, max_rows=300)
        assert got[280, 1].isnan().all() and got[290, 0].isnan().all()
        got[280, 1], got[290, 0] = y[280, 1], y[290, 0]
        off = np.abs(got.double().cpu().numpy() - want)
        assert (off <= lim).all()
        c.backend.device_status()
        c.v_exp.copy_(torch.from_numpy(rng.integers(90, 150, c.v_exp.shape).astype(np.uint8)))
