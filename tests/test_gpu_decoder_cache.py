"""Qwen3-shaped decoders that keep their keys and values in 8 bits, and the log probabilities of given tokens, against a numpy
restatement that quantizes where they quantize."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nn_b200 import api, decoder, kv_cache
from nn_b200.formats import QuantFormat as Q
from oracle import qwen3_ref as ref
from tests import kv_reference as kvref
from tests import test_gpu_fused_step as fused

pytestmark = pytest.mark.gpu
HIDDEN, FFN, VOCAB, EPS = 128, 192, 160, 1e-6


@pytest.fixture
def f32_products():
    """Products of more than 16 rows round their operands to bf16 (a bar of 1e-2); with f32 operands what is left is the cache's."""
    b = api.gpu_backend()
    b.set_path(api.PATH_F32)
    yield
    b.set_path(api.PATH_AUTO)


def _decoder(group, max_seq, act_dtype=api.F32, seed=0):
    rng = np.random.default_rng(seed + group)
    kv = 2
    cfg = decoder.DecoderConfig(hidden=HIDDEN, n_heads=kv * group, n_kv_heads=kv, ffn=FFN, n_layers=2, vocab=VOCAB, max_seq=max_seq, act_dtype=act_dtype)
    b = api.gpu_backend()
    dec = decoder.Decoder(b, cfg)

    def weight(n, k):
        w = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32) / np.sqrt(k).astype(np.float32)).to(torch.bfloat16).cuda()
        return api.DeviceWeight.from_device(b, Q.BF16_DENSE, w.view(torch.uint8).reshape(-1), n, k), w.double().cpu().numpy()

    norm = lambda n: (1.0 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
    model = {"layers": [], "cfg": cfg}
    q, k = cfg.n_heads * 128, kv * 128
    for i in range(cfg.n_layers):
        ws = [weight(n, m) for n, m in ((q, HIDDEN), (k, HIDDEN), (k, HIDDEN), (HIDDEN, q), (FFN, HIDDEN), (FFN, HIDDEN), (HIDDEN, FFN))]
        ns = [norm(HIDDEN), norm(HIDDEN), norm(128), norm(128)]
        dec.set_layer(i, *[w for w, _ in ws], *ns)
        model["layers"].append(([f for _, f in ws], ns))
    embed = torch.from_numpy(rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32)).to(torch.bfloat16).cuda()
    head, model["head"] = weight(VOCAB, HIDDEN)
    model["embed"], model["final"] = embed.double().cpu().numpy(), norm(HIDDEN)
    dec.set_head(embed, model["final"], head)
    return dec, model


class Restated:
    """The decoder in 64 bits with its caches: keys and values quantized portion by portion."""

    def __init__(self, model, fmt, block):
        c = model["cfg"]
        self.model, self.fmt, self.block, self.pos = model, fmt, block, 0
        blocks = -(-c.max_seq // block)
        self.k = [(np.zeros((blocks, c.n_kv_heads, block, 128)), np.full((blocks, c.n_kv_heads), 7, np.uint8)) for _ in model["layers"]]
        self.v = [(np.zeros((blocks, c.n_kv_heads, block, 128)), np.full((blocks, c.n_kv_heads), 7, np.uint8)) for _ in model["layers"]]
        self.rope = [t.astype(np.float64) for t in ref.rope_tables(128, c.max_seq, c.rope_theta)]

    def rows(self, ids):
        c, n, p0 = self.model["cfg"], len(ids), self.pos
        cos, sin = (t[p0:p0 + n, None] for t in self.rope)
        h = self.model["embed"][ids]
        rms = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w  # noqa: E731
        rot = lambda x: np.concatenate([x[..., :64] * cos - x[..., 64:] * sin, x[..., :64] * sin + x[..., 64:] * cos], -1)  # noqa: E731
        slots = list(range(p0, p0 + n))
        for l, ((q, k, v, o, g, u, d), (n1, n2, nq, nk)) in enumerate(self.model["layers"]):
            x = rms(h, n1)
            Q_, K, V = (x @ q.T).reshape(n, -1, 128), (x @ k.T).reshape(n, -1, 128), (x @ v.T).reshape(n, -1, 128)
            Q_, K = rot(rms(Q_, nq)), rot(rms(K, nk))
            for (vals, exps), rows in ((self.k[l], K), (self.v[l], V)):
                kvref.append(self.fmt, vals, exps, rows, slots, self.block)
            y, _, _ = kvref.attend(Q_, self.k[l][0], self.v[l][0], [list(range(len(self.k[l][0])))], [p0 + n], [0, n], self.block, 128 ** -0.5, 0)
            h = h + y.reshape(n, -1) @ o.T
            x = rms(h, n2)
            gate = x @ g.T
            h = h + (gate / (1 + np.exp(-gate)) * (x @ u.T)) @ d.T
        self.pos += n
        return rms(h, self.model["final"]) @ self.model["head"].T


@pytest.mark.parametrize("fmt", [kv_cache.INT8, kv_cache.E4M3])
@pytest.mark.parametrize("group,block", [(1, 16), (4, 32), (8, 256)])
@pytest.mark.parametrize("count", [2, 19, 75])
def test_prompts_and_steps_over_an_8_bit_cache(f32_products, fmt, group, block, count):
    """f32 decoders: the bar of their logits, 2e-3. A key or value at the border of two codes may take the other one, which is within it."""
    dec, model = _decoder(group, count + 6)
    dec.set_cache(fmt, block)
    want, ids = Restated(model, fmt, block), np.random.default_rng(count).integers(0, VOCAB, count + 4)
    cut = count * 2 // 3
    for a, e in ((0, cut), (cut, count)) + tuple((count + i, count + i + 1) for i in range(4)):
        if e == a:
            continue
        got = dec.extend(ids[a:e], a, list(range(e - a)))
        exact = want.rows(ids[a:e])
        assert np.abs(got - exact).max() <= 2e-3 * np.abs(exact).max(), (a, e, np.abs(got - exact).max() / np.abs(exact).max())
    k, v, ke, ve = dec.cache(1)
    for codes, exps, (vals, e) in ((k, ke, want.k[1]), (v, ve, want.v[1])):
        got = kvref.decode(fmt, codes.cpu().numpy(), exps.cpu().numpy()).transpose(0, 2, 1, 3).reshape(-1, 2, 128)[:count + 4]
        exact = vals.transpose(0, 2, 1, 3).reshape(-1, 2, 128)[:count + 4]
        assert np.mean(got != exact) <= 1e-3   # codes next to a border
    assert dec.buffers()[0] is None
    dec.backend.device_status()
    dec.release()


@pytest.mark.parametrize("act_dtype", [api.F32, api.BF16])
def test_generation_replayed_from_a_graph_and_again(act_dtype):
    """The same tokens with and without a graph, after another sequence, and from a restart in the middle."""
    prompt = np.random.default_rng(3).integers(0, VOCAB, 37).tolist()
    out = []
    for use_graph in (True, False):
        dec, _ = _decoder(4, 128, act_dtype)
        dec.set_cache(kv_cache.INT8, 16)
        first = dec.complete(prompt, 60, use_graph)
        dec.complete(prompt[:5], 30, use_graph)
        assert dec.complete(prompt, 60, use_graph) == first
        dec.prefill(prompt[20:], 20)            # the positions from 20 on again
        assert dec.state()[:2] == (first[0], 37)
        assert dec.generate(first[0], 37, 20, use_graph) == first[1:21]
        out.append(first)
        dec.backend.device_status()
        dec.release()
    assert out[0] == out[1]


@pytest.mark.parametrize("fmt", [kv_cache.INT8, kv_cache.E4M3])
@pytest.mark.parametrize("heads,kv", [(2, 2), (16, 8), (16, 2)])
def test_fused_steps_over_an_8_bit_cache(fmt, heads, kv):
    """A bf16 decoder of Q4_K weights, whose step keeps norms, activation and residual sums in the products' kernels, against the step
    with kernels of their own: 1e-2 in the 2-norm as with an f32 cache. A difference d of a new key or value may also turn its code by a
    step s, which adds d s to its mean square: d = 2^-9 and s = 2^-6 of the largest value, elements of a third of it, sqrt(d s) * 3 =
    1.7e-2 where the new token is all there is, 1.7e-2 / sqrt(16) behind 15 others."""
    dec, b = fused._model(heads, kv, 2, 600), api.gpu_backend()
    dec.set_cache(fmt, 32)
    logits, caches = dec.buffers()[2], [dec.cache(i) for i in range(2)]
    g = torch.Generator(device="cuda").manual_seed(5)
    past = [[torch.randint(0, 120, t.shape, device="cuda", generator=g, dtype=torch.uint8) if t.dim() == 4 else torch.full_like(t, 121) for t in c] for c in caches]
    for at in (0, 1, 15, 32, 599):
        got = []
        for path in (api.PATH_AUTO, api.PATH_SKINNY):
            for c, old in zip(caches, past):
                for t, o in zip(c, old):
                    t.copy_(o)
            b.set_path(path)
            try:
                dec.reset(7, at)
                before = b.launch_count()
                dec.step()
                launches = b.launch_count() - before
            finally:
                b.set_path(api.PATH_AUTO)
            torch.cuda.synchronize()
            b.device_status()
            got.append((launches, logits[:].clone()))
        assert got[0][0] < got[1][0]   # (the fused step is what ran)
        assert float((got[0][1] - got[1][1]).norm() / got[1][1].norm()) < 1e-2 + 1.7e-2 / (at + 1) ** 0.5, at
    dec.release()


def test_the_end_of_the_context_with_an_8_bit_cache():
    dec, _ = _decoder(2, 33)
    dec.set_cache(kv_cache.E4M3, 16)
    dec.reset(3, 30)
    for _ in range(3):
        dec.step()
    with pytest.raises(api.Unsupported):
        dec.step()
    dec.backend.device_status()
    stream = torch.cuda.Stream()
    dec.reset(3, 31, stream)
    with torch.cuda.stream(stream):
        dec.step(stream)
        stream.synchronize()
        dec.reset(3, 31, stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            dec.step(torch.cuda.current_stream())
        for _ in range(4):
            g.replay()
    stream.synchronize()
    with pytest.raises(api.Unsupported):
        dec.backend.device_status(stream)
    # the decoder serves another sequence afterwards
    a = dec.complete([1, 2, 3], 8)
    assert a == dec.complete([1, 2, 3], 8)
    dec.backend.device_status()
    dec.release()


def test_caches_that_a_decoder_refuses():
    dec, _ = _decoder(1, 64)
    for args in ((2, 16), (0, 24), (0, 512), (-1, 16)):
        with pytest.raises(api.TensorError):
            dec.set_cache(*args)
    with pytest.raises(api.Unsupported):
        dec.cache(0)
    dec.set_cache(0, 16)
    with pytest.raises(api.Unsupported):
        dec.set_cache(0, 16)
    with pytest.raises(api.InvalidArgument):
        dec.cache(2)
    dec.release()
    dec, _ = _decoder(1, 64)
    dec.prefill([1, 2, 3])
    with pytest.raises(api.Unsupported):
        dec.set_cache(0, 16)
    dec.release()
    block = decoder.BlockDecoder(api.gpu_backend(), hidden=64, vocab=32, blocks=[decoder.BlockConfig(heads=1, kv_heads=1, dim=64, vdim=64)], max_seq=16)
    with pytest.raises(api.Unsupported):
        block.set_cache(0, 16)
    block.release()


@pytest.mark.parametrize("cache", [None, kv_cache.INT8])
@pytest.mark.parametrize("count", [1, 2, 64, 65, 150])
def test_scores_of_given_tokens(cache, count):
    """Against the logits of `extend` on the same decoder: the bounds of the log probabilities alone."""
    dec, _ = _decoder(2, 200)
    if cache is not None:
        dec.set_cache(cache)
    ids = np.random.default_rng(count).integers(0, VOCAB, count)
    logits = dec.extend(ids, 0, list(range(count)))
    r = dec.score(ids, 0, top=7)
    given = np.append(ids[1:], 0)
    lp, ent, order, tl = kvref.logprobs(logits, given, 7)
    assert r.logprob[-1] == 0 and np.abs(r.logprob[:-1] - lp[:-1]).max(initial=0) <= 1e-5 and np.abs(r.entropy - ent).max() <= 1e-5
    assert np.array_equal(r.top_tokens, order) and np.abs(r.top_logprobs - tl).max() <= 1e-5
    # behind given tokens, and without alternatives
    at = dec.state()[1]
    more = dec.score([5, 6, 7], at, given=[6, -1, 9])
    assert more.top_tokens is None and more.logprob[1] == 0 and (more.logprob[[0, 2]] < 0).all()
    dec.release()


def test_scores_that_are_refused():
    dec, _ = _decoder(1, 32)
    for args, kw in ((([1, 2],), dict(given=[3, VOCAB])), (([1, 2],), dict(top=33)), (([1, 2],), dict(top=-1)), (([1, VOCAB],), {}), (([1, 2],), dict(given=[1])),
                     ((list(range(40)),), {})):
        with pytest.raises((api.TensorError, ValueError)):
            dec.score(*args, **kw)
    assert dec.score([1, 2]).logprob.shape == (2,)
    dec.release()


def test_scores_of_a_block_decoder():
    blocks = [decoder.BlockConfig(heads=2, kv_heads=1, dim=64, vdim=64, ffn=128, rot_dims=64, scale=0.125)]
    dec = decoder.BlockDecoder(api.gpu_backend(), hidden=128, vocab=96, blocks=blocks, max_seq=64, act_dtype=api.F32)
    rng = np.random.default_rng(1)
    bits = lambda n, k: (torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32)) / np.sqrt(k)).to(torch.bfloat16).view(torch.uint16).numpy()  # noqa: E731
    dec.set_block(0, decoder.BlockTensors(norm=np.ones(128, np.float32), q=bits(128, 128), k=bits(64, 128), v=bits(64, 128), o=bits(128, 128), gate=bits(128, 128), up=bits(128, 128),
                                          down=bits(128, 128)))
    e = bits(96, 128)
    dec.set_head(e, np.ones(128, np.float32), e)
    ids = rng.integers(0, 96, 20)
    logits = dec.extend(ids, 0, list(range(20)))
    r = dec.score(ids, 0, top=3)
    lp, ent, order, _ = kvref.logprobs(logits, np.append(ids[1:], 0), 3)
    assert np.abs(r.logprob[:-1] - lp[:-1]).max() <= 1e-5 and np.abs(r.entropy - ent).max() <= 1e-5 and np.array_equal(r.top_tokens, order)
    dec.release()


@pytest.mark.parametrize("fmt,block", [(kv_cache.INT8, 32), (kv_cache.E4M3, 64)])
@pytest.mark.parametrize("group", [1, 4])
def test_long_prompts_over_an_8_bit_cache(f32_products, fmt, block, group):
    """Prompts of several tiles of the prompt attention's, in two portions, the second far behind the first one's start."""
    count, cut = 640, 411
    dec, model = _decoder(group, count + 2)
    dec.set_cache(fmt, block)
    want, ids = Restated(model, fmt, block), np.random.default_rng(group).integers(0, VOCAB, count + 2)
    for a, e in ((0, cut), (cut, count), (count, count + 1), (count + 1, count + 2)):
        got, exact = dec.extend(ids[a:e], a, list(range(e - a))), want.rows(ids[a:e])
        assert np.abs(got - exact).max() <= 2e-3 * np.abs(exact).max(), (a, e, np.abs(got - exact).max() / np.abs(exact).max())
    dec.backend.device_status()
    dec.release()
