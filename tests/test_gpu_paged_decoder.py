"""GPU: several sequences at once over the paged 4-bit KV cache (moty_b200.decoder.PagedDecoder): prompts of different
length in one batch, single tokens, forks, ended sequences, compaction, a captured decode loop -- against the CPU oracle's
products composed with an attention over rows quantised by the cache's rule."""
import numpy as np
import pytest

from test_gpu_decoder import _rmsnorm
from test_gpu_kv4 import quant

pytestmark = pytest.mark.gpu


def _model(gpu, rng, H, KV, hd, D, I, V, NL, fused):
    raw = lambda O, K: (rng.integers(-127, 128, (O, K), dtype=np.int8), rng.uniform(0.0005, 0.0015, O).astype(np.float32))
    W = dict(layers=[], final_norm=rng.uniform(0.5, 1.5, D).astype(np.float32))
    W["head"] = (rng.integers(-127, 128, (V, D), dtype=np.int8), rng.uniform(0.005, 0.015, V).astype(np.float32))
    from moty_b200.decoder import DenseLayer
    layers = []
    for _ in range(NL):
        l = {n: raw(*s) for n, s in (("q", (H * hd, D)), ("k", (KV * hd, D)), ("v", (KV * hd, D)), ("o", (D, H * hd)), ("gate", (I, D)),
                                     ("up", (I, D)), ("down", (D, I)))}
        l.update({n: rng.uniform(0.5, 1.5, s).astype(np.float32) for n, s in (("in_ln", D), ("post_ln", D), ("qn", hd), ("kn", hd))})
        W["layers"].append(l)
        m = {n: gpu.Mat.i8(*l[n]) for n in ("q", "k", "v", "o", "gate", "up", "down")}
        qkv = gpu.Mat.i8(np.concatenate([l[n][0] for n in "qkv"]), np.concatenate([l[n][1] for n in "qkv"])) if fused else None
        layers.append(DenseLayer(m["q"], m["k"], m["v"], m["o"], m["gate"], m["up"], m["down"], l["in_ln"], l["post_ln"], l["qn"], l["kn"], qkv=qkv))
    return W, layers, gpu.Mat.i8(*W["head"])


class _Plain:
    """One sequence on the CPU: the oracle's products; norm, rotation, quantised rows and softmax in numpy."""

    def __init__(self, oracle, W, H, KV, hd):
        self.o, self.W, self.H, self.KV, self.hd = oracle, W, H, KV, hd
        self.k = [np.zeros((0, KV, hd)) for _ in W["layers"]]; self.v = [np.zeros((0, KV, hd)) for _ in W["layers"]]

    def copy(self):
        c = _Plain(self.o, self.W, self.H, self.KV, self.hd)
        c.k, c.v = list(self.k), list(self.v)
        return c

    def _rope(self, x, pos):
        half = self.hd // 2
        j = np.arange(half, dtype=np.float32)
        ang = (np.float32(pos) / np.power(np.float32(1e6), 2 * j / np.float32(self.hd), dtype=np.float32)).astype(np.float32)
        c, s = np.cos(ang), np.sin(ang)
        lo, hi = x[..., :half], x[..., half:]
        return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1).astype(np.float32)

    def step(self, ids):
        o, W = self.o, self.W
        hq, hs = W["head"]
        x = np.stack([hs[i] * hq[i].astype(np.float32) for i in ids]).astype(np.float32)
        S, T0 = len(ids), self.k[0].shape[0]
        for n, l in enumerate(W["layers"]):
            h = _rmsnorm(x, l["in_ln"], 1e-6)
            q, k, v = (o.matmul_q_s(h, *l[m]) for m in ("q", "k", "v"))
            norm = lambda a, w: _rmsnorm(a.reshape(-1, self.hd), w, 1e-6).reshape(S, -1, self.hd)
            q, k = norm(q, l["qn"]), norm(k, l["kn"])
            q = np.stack([self._rope(q[s], T0 + s) for s in range(S)]); k = np.stack([self._rope(k[s], T0 + s) for s in range(S)])
            self.k[n] = np.concatenate([self.k[n], quant(k)[0]]); self.v[n] = np.concatenate([self.v[n], quant(v.reshape(S, self.KV, self.hd))[0]])
            ctx = np.zeros((S, self.H, self.hd))
            for s in range(S):
                for a in range(self.H):
                    g = a // (self.H // self.KV)
                    sc = self.k[n][:T0 + s + 1, g] @ q[s, a].astype(np.float64) / np.sqrt(self.hd)
                    w = np.exp(sc - sc.max())
                    ctx[s, a] = w @ self.v[n][:T0 + s + 1, g] / w.sum()
            x = x + o.matmul_q_s(ctx.astype(np.float32).reshape(S, -1), *l["o"])
            h = _rmsnorm(x, l["post_ln"], 1e-6)
            x = x + o.matmul_q_s(o.silu_mul(o.matmul_q_s(h, *l["gate"]), o.matmul_q_s(h, *l["up"])), *l["down"])
        return o.matmul_q_s(_rmsnorm(x[-1:], W["final_norm"], 1e-6), hq, hs)[0]


# Logits: the activation rows between the products are re-quantised to int8 (one code is 1/127 of a row's largest value) and
# key and value rows to 4 bits, so a difference in the last bit of a cosine can move a code by one.  A moved activation code
# changes a product by 1/127 of one of its ~D terms, a moved 4-bit code one of the T x hd cached values by 1/7 of its
# group's largest; with D >= 256 terms of random sign and a handful of codes moved per step, that is below
# 2 (1/127) / sqrt(256) + 2 (1/7) / sqrt(40 * 32) = 0.009 of the logits' size: 0.02 leaves a factor of two.
TOL = 0.02


def _agree(got, want):
    size = np.abs(want).max()
    err = np.abs(got - want).max() / size
    assert err <= TOL, f"logits off by {err:.3g} of their size"
    # the pick: the reference's, or one within the tolerance of it
    assert want[int(np.argmax(got))] >= want.max() - 2 * TOL * size


@pytest.mark.parametrize("H,KV,hd,fused", [(8, 4, 32, False), (8, 2, 64, True), (4, 4, 96, True)])
def test_a_run_of_sequences(gpu, oracle, H, KV, hd, fused):
    rng = np.random.default_rng(H * hd)
    D, I, V, NL = 256, 512, 1000, 2
    from moty_b200.decoder import PagedDecoder
    W, layers, head = _model(gpu, rng, H, KV, hd, D, I, V, NL, fused)
    dec = PagedDecoder(layers, head, W["final_norm"], H, KV, hd, pages=14, max_seqs=6, max_pages=4, theta=1e6, max_S=16)
    plain, toks = {}, {}

    def feed(batch):
        out, lg = dec.run(batch, want_logits=True)
        for i, (s, ids) in enumerate(batch):
            want = plain[s].step(list(ids))
            _agree(lg[i], want)
            assert out[i] == int(np.argmax(lg[i]))
            toks[s] = int(out[i])

    a, b, c = dec.new(), dec.new(), dec.new()
    for s in (a, b, c):
        plain[s] = _Plain(oracle, W, H, KV, hd)
    feed([(a, rng.integers(0, V, 70)), (b, rng.integers(0, V, 1)), (c, rng.integers(0, V, 40))])
    feed([(c, [toks[c]]), (a, [toks[a]])])                          # single tokens, another order, one left out
    feed([(b, rng.integers(0, V, 30)), (a, [toks[a]]), (c, [toks[c]])])        # a prompt block beside single tokens
    # forks share what is there and go their own ways
    f1, f2 = dec.fork(a, 2)
    for f in (f1, f2):
        plain[f] = plain[a].copy()
    free = dec.kv.free_pages()
    feed([(a, [5]), (f1, [6]), (f2, [7]), (b, [toks[b]])])
    assert dec.kv.free_pages() == free and len({toks[a], toks[f1], toks[f2]}) >= 1
    # end one, compact, go on
    dec.end(c); del plain[c]
    moved = dec.compact()
    live = np.unique(dec.table[dec.table >= 0])
    assert live.max() == live.size - 1 and moved > 0
    feed([(f2, [toks[f2]]), (b, [toks[b]]), (a, [toks[a]]), (f1, [toks[f1]])])
    # a captured loop equals steps one by one
    g = dec.greedy([a, f1], [toks[a], toks[f1]], 5)
    for i, s in enumerate((a, f1)):
        for n in range(5):
            tok = toks[s] if n == 0 else int(g[i, n - 1])
            lg = plain[s].step([tok])
            assert lg[int(g[i, n])] >= lg.max() - 2 * TOL * np.abs(lg).max()
    # refusals leave everything as it was
    before, lens = dec.table.copy(), dec.lens.copy()
    for bad in ([(a, [1]), (a, [2])], [(c, [1])], [(a, [])], [(a, rng.integers(0, V, 300))], [(99, [1])]):
        with pytest.raises(gpu.MotyCudaError):
            dec.run(bad)
    with pytest.raises(gpu.MotyCudaError):
        dec.fork(a, 5)
    assert np.array_equal(before, dec.table) and np.array_equal(lens, dec.lens)
    for s in list(plain):
        dec.end(s)
    assert dec.kv.free_pages() == 14
    dec.close()


def test_replayed_loop_equals_steps(gpu):
    """The captured loop and token-by-token runs give the same ids (the same kernels on the same rows), single and forked."""
    rng = np.random.default_rng(3)
    H, KV, hd, V = 8, 2, 64, 1000
    from moty_b200.decoder import PagedDecoder
    W, layers, head = _model(gpu, rng, H, KV, hd, 256, 512, V, 3, True)
    dec = PagedDecoder(layers, head, W["final_norm"], H, KV, hd, pages=40, max_seqs=4, max_pages=8)
    prompts = [rng.integers(0, V, n) for n in (100, 7, 64)]
    sids = [dec.new() for _ in prompts]
    first = dec.run(list(zip(sids, prompts)))
    g = dec.greedy(sids, first, 70)                                 # over a page's end
    for s in sids:
        dec.end(s)
    sids = [dec.new() for _ in prompts]
    tok = dec.run(list(zip(sids, prompts)))
    assert np.array_equal(tok, first)
    one = []
    for _ in range(70):
        tok = dec.run([(s, [t]) for s, t in zip(sids, tok)])
        one.append(tok)
    assert np.array_equal(np.array(one).T, g)
    dec.close()


def test_forks_and_tokens_that_are_none(gpu):
    rng = np.random.default_rng(4)
    from moty_b200.decoder import PagedDecoder
    W, layers, head = _model(gpu, rng, 4, 2, 32, 128, 256, 300, 1, True)
    dec = PagedDecoder(layers, head, W["final_norm"], 4, 2, 32, pages=8, max_seqs=3, max_pages=4)
    s = dec.new()
    dec.run([(s, rng.integers(0, 300, 70))])
    table, lens, free = dec.table.copy(), dec.lens.copy(), dec.kv.free_pages()
    for bad in (lambda: dec.fork(s, 0), lambda: dec.fork(s, -1), lambda: dec.run([(s, [300])]), lambda: dec.run([(s, [5, -1])]),
                lambda: dec.run([(s, [])]), lambda: dec.greedy([s], [300], 3), lambda: dec.greedy([s], [1, 2], 3), lambda: dec.greedy([s], [1], 0)):
        with pytest.raises(gpu.MotyCudaError):
            bad()
        assert np.array_equal(table, dec.table) and np.array_equal(lens, dec.lens) and dec.kv.free_pages() == free
    dec.close()
