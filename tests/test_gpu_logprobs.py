"""Log probabilities, entropies and most probable tokens of rows of logits against 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nn_b200 import api
from nn_b200.logprobs import token_logprobs
from tests import kv_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(x, tokens, top):
    """lse = m + ln l: an exponent is off by 2^-22 relative and its argument by 2^-24 of itself, a thread's sums round by 2^-24 per
    element (one in 512 of the row), differences to the maximum by 2^-24 of their size. Entropy: the same on numbers of its size."""
    r = token_logprobs(x, tokens, top)
    lp, ent, order, tl = ref.logprobs(x.double().cpu().numpy(), tokens.cpu().numpy(), top)
    eps = 2.0 ** -20 + (x.shape[1] / 512 + 64) * 2.0 ** -24
    spread = 1 + np.log(x.shape[1])
    assert (np.abs(r.logprob.double().cpu().numpy() - lp) <= eps * spread + 2.0 ** -22 * np.abs(lp)).all()
    assert (np.abs(r.entropy.double().cpu().numpy() - ent) <= 2 * eps * spread).all()
    if top:
        assert np.array_equal(r.top_tokens.cpu().numpy(), order)
        assert (np.abs(r.top_logprobs.double().cpu().numpy() - tl) <= eps * spread + 2.0 ** -22 * np.abs(tl)).all()
    return r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 31), (2, 100), (5, 1000), (1, 4097), (1, 151936), (7, 32001), (160, 9001), (400, 515)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows_of_every_size(dtype, rows, vocab, top):
    g = torch.Generator(device=DEV).manual_seed(vocab + top)
    x = (torch.randn(rows, vocab, device=DEV, generator=g) * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,), device=DEV, generator=g, dtype=torch.int32)
    check(x, t, min(top, vocab))
    api.gpu_backend().device_status()


@pytest.mark.parametrize("vocab", [700, 40000])
def test_orders_and_equal_values(vocab):
    i = torch.arange(vocab, device=DEV, dtype=torch.float32)
    rows = [i / vocab * 20, -i / vocab * 20, torch.zeros_like(i), (i % 3), -(i % 7), torch.where(i == vocab - 1, 5.0, 0.0), torch.where(i < 20, 1.0, -60.0), i * 0 - 0.0]
    x = torch.stack(rows)
    x[7, ::2] = 0.0   # 0 and -0 are equal
    t = torch.tensor([0, vocab - 1, 5, 7, 100, vocab - 1, 3, 9], device=DEV)
    for top in (1, 7, 32):
        check(x, t, top)


def test_large_small_and_shifted_logits():
    x = torch.randn(6, 5001, device=DEV)
    x[0] += 5000
    x[1] -= 5000
    x[2] *= 300
    x[3] *= 1e-30
    x[4] = 1e30 * torch.sign(x[4])
    x[5, 17] = 200
    t = torch.full((6,), 17, device=DEV)
    r = check(x[[0, 1, 2, 3, 5]], t[:5], 8)
    assert r.entropy.isfinite().all()
    r = token_logprobs(x[4:5], t[:1], 4)
    assert r.logprob.item() <= 0 and torch.equal(r.top_tokens[0].long(), (x[4] > 0).nonzero()[:4, 0])


@pytest.mark.parametrize("vocab", [50, 20000])
def test_logits_of_minus_infinity(vocab):
    x = torch.randn(4, vocab, device=DEV)
    x[0, 1:] = -float("inf")          # one token left
    x[1, ::2] = -float("inf")
    x[2] = -float("inf")              # none
    x[3, 5:] = torch.finfo(torch.float32).min
    t = torch.tensor([0, 0, 3, 7], device=DEV)
    r = token_logprobs(x, t, 6)
    lp, ent, order, tl = (a[[0, 1, 3]] for a in ref.logprobs(x.double().cpu().numpy(), t.cpu().numpy(), 6))
    keep = [0, 1, 3]
    got = r.top_logprobs.double().cpu().numpy()[keep]
    assert np.array_equal(r.top_tokens.cpu().numpy()[keep], order)
    assert np.allclose(r.logprob.double().cpu().numpy()[keep], lp, rtol=1e-6, atol=1e-5) and np.allclose(r.entropy.double().cpu().numpy()[keep], ent, atol=1e-5)
    assert np.allclose(got, tl, rtol=1e-6, atol=1e-5)
    assert r.logprob[2] == -float("inf") and r.entropy[2] == 0 and (r.top_logprobs[2] == -float("inf")).all() and r.top_tokens[2].tolist() == list(range(6))


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("vocab,at", [(40, 3), (30000, 0), (30000, 29999)])
def test_rows_with_numbers_that_are_not_finite(what, vocab, at):
    x = torch.randn(3, vocab, device=DEV)
    clean = token_logprobs(x, torch.zeros(3, device=DEV, dtype=torch.int32), 4)
    x[1, at] = what
    r = token_logprobs(x, torch.zeros(3, device=DEV, dtype=torch.int32), 4)
    assert r.entropy[1].isnan() and r.top_tokens[1, 0] == at
    assert r.logprob[1].isnan() or (what > 0 and at != 0)
    for a, b in ((clean.logprob, r.logprob), (clean.entropy, r.entropy), (clean.top_tokens, r.top_tokens), (clean.top_logprobs, r.top_logprobs)):
        assert torch.equal(a[[0, 2]], b[[0, 2]])


def test_tokens_that_are_none_and_beyond():
    x = torch.randn(3, 100, device=DEV)
    r = token_logprobs(x, torch.tensor([-1, -100, 5], device=DEV))
    assert r.logprob[0] == 0 and r.logprob[1] == 0 and r.top_tokens is None
    api.gpu_backend().device_status()
    r = token_logprobs(x, torch.tensor([100, 2 ** 40, 5], device=DEV))
    assert r.logprob[0].isnan() and r.logprob[1].isnan() and r.logprob[2].isfinite()
    with pytest.raises(api.InvalidArgument):
        api.gpu_backend().device_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_lie_apart_or_off_their_boundaries(dtype):
    base = (torch.randn(6, 5003, device=DEV) * 2).to(dtype)
    t = torch.tensor([1, 2, 3, 4, 5, 6], device=DEV)
    for lo, hi in ((1, 5003), (3, 4100), (7, 4999), (0, 5003)):
        check(base[:, lo:hi], t, 9)
    check(base.t().contiguous().t(), t, 9)
    check(base[:1].expand(6, 5003), t, 3)
    check(base[::2], t[:3], 3)
    check(base.half() if dtype == torch.float32 else base.double(), t, 3)


def test_the_same_bits_every_time_and_on_another_stream():
    x = torch.randn(3, 60000, device=DEV)
    t = torch.tensor([5, 6, 7], device=DEV, dtype=torch.int32)
    want = token_logprobs(x, t, 32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = token_logprobs(x, t, 32)
        for _ in range(5):
            g.replay()
    torch.cuda.synchronize()
    for name in ("logprob", "entropy", "top_tokens", "top_logprobs"):
        assert torch.equal(getattr(want, name), getattr(got, name))


def test_many_rows():
    check(torch.randn(70001, 33, device=DEV), torch.zeros(70001, device=DEV, dtype=torch.int32), 3)


def test_wrong_tensors_are_refused():
    x, t = torch.zeros(2, 10, device=DEV), torch.zeros(2, device=DEV, dtype=torch.int32)
    for args in ((x[0], t), (x, t[:1]), (x.cpu(), t), (x, t.cpu()), (x, t, 11), (x, t, -1), (torch.zeros(2, 100, device=DEV), t, 33)):
        with pytest.raises(api.TensorError):
            token_logprobs(*args)
    assert token_logprobs(x[:0], t[:0], 2).top_tokens.shape == (0, 2)


def test_two_threads_with_other_vocabularies():
    """Two contexts in two threads, one with a large vocabulary, the other with a small one, call after call."""
    import threading

    x = {v: torch.randn(1, v, device=DEV) for v in (151936, 60000)}
    t = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = {v: token_logprobs(x[v], t, 5) for v in x}
    torch.cuda.synchronize()
    wrong = []

    def work(v):
        b = api.Backend()
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    r = token_logprobs(x[v], t, 5, b)
                torch.cuda.current_stream().synchronize()
            if not (torch.equal(r.logprob, want[v].logprob) and torch.equal(r.top_tokens, want[v].top_tokens)):
                wrong.append(v)
        except Exception as e:   # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(v,)) for v in x]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def masked_rows(rows, vocab, allowed, dtype, seed=0):
    """Logits of a grammar: all but `allowed` tokens of a row are -inf."""
    rng = np.random.default_rng(seed + vocab + allowed)
    x = np.full((rows, vocab), -np.inf, np.float32)
    for r in range(rows):
        at = rng.choice(vocab, allowed, replace=False)
        x[r, at] = rng.standard_normal(allowed) * 3
    return torch.from_numpy(x).to("cuda:0", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (3, 32003), (5, 700), (300, 5001)])
@pytest.mark.parametrize("allowed", [1, 5, 20, 31, 33, 200])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_alternatives_where_few_tokens_are_allowed(dtype, rows, vocab, allowed, top):
    """Those that are allowed, then the lowest of the others at -inf."""
    x = masked_rows(rows, vocab, allowed, dtype)
    x[0, :3] = -float("inf")
    if rows > 1:
        x[1, :3], x[-1, -2:] = 1.5, 2.5   # next to the slice's edges
    if not x.isfinite().any(1).all():
        x[0, 3] = 0.5
    token = x.float().argmax(1)
    lp, ent, order, tl = ref.logprobs(x.double().cpu().numpy(), token.cpu().numpy(), top)
    r = token_logprobs(x, token, top)
    assert np.array_equal(r.top_tokens.cpu().numpy(), order)
    got, there = r.top_logprobs.double().cpu().numpy(), np.isfinite(tl)
    lim = (2.0 ** -20 + (vocab / 512 + 64) * 2.0 ** -24) * (1 + np.log(vocab))   # (as in `check`)
    assert (got[~there] == -np.inf).all() and (np.abs(got[there] - tl[there]) <= lim + 2.0 ** -22 * np.abs(tl[there])).all()
    assert (np.abs(r.logprob.double().cpu().numpy() - lp) <= lim + 2.0 ** -22 * np.abs(lp)).all()
    assert (np.abs(r.entropy.double().cpu().numpy() - ent) <= 2 * lim).all()


def test_masked_rows_cost_what_others_do():
    """They are not read again for every alternative."""
    x = torch.randn(64, 151936, device="cuda:0")
    few = masked_rows(64, 151936, 20, torch.float32)
    token = torch.zeros(64, dtype=torch.int32, device="cuda:0")

    def shortest(t):
        best = 1e9
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                token_logprobs(t, token, 20)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    plain, masked = shortest(x), shortest(few)
    print(f"{plain * 200:.1f} and {masked * 200:.1f} us")
    assert masked <= 3 * plain


def test_logits_beyond_32_bits_of_bytes():
    x = torch.zeros(9001, 128001, device="cuda:0")   # 4.6 GB
    x[-1].normal_()
    token = torch.full((9001,), 77, dtype=torch.int32, device="cuda:0")
    r, one = token_logprobs(x, token, 3), token_logprobs(x[-1:].clone(), token[-1:], 3)
    assert torch.equal(r.top_tokens[-1], one.top_tokens[0]) and float((r.logprob[-1] - one.logprob[0]).abs()) <= 1e-5
    assert r.top_tokens[-2].tolist() == [0, 1, 2] and abs(float(r.logprob[0]) + np.log(128001)) <= 1e-5
