"""GPU: the paged 4-bit KV cache -- store and fetch bit for bit, attention against a 64-bit implementation, forks,
compaction, batches that are none, graphs, streams, and a run of them together.

Tolerance of the attention (tol): with e = 2^-24 (half a step of f32),
  * a query value reaches the products as two 11-bit pieces, 2^-23 relative at worst, a key value exactly; the hd products
    are added in f32 in some order, and the matrix unit may cut a sum off instead of rounding it (2 e a step):
        |ds| <= (2 e + 2 e (hd / 16 + 16) + 4 e) A,   A = max_t scale sum_d |q_d k_td|
    (4 e: the scale, the difference to the maximum and the base-2 argument); exp adds 2^-22 = 4 e relative;
  * weights times steps reach the second product with 2^-23 relative; sums over T positions run in tiles of 16, so a term
    passes at most T / 16 + 64 additions (the last 64: tile, warp and split joins), 2 e each, in numerator and denominator.
  |dctx| <= V (2 |ds| + 8 e + 2 * 2 e (T / 16 + 64)),   V = max_t |v_t| over the positions seen.
"""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(scope="module")
def t():
    import torch
    torch.backends.cuda.matmul.allow_tf32 = False
    return torch


def quant(x):
    """numpy: (values f64, codes, steps f16) of rows x [..][hd] f32, by the definition."""
    x = np.asarray(x, np.float32)
    v = x.reshape(*x.shape[:-1], -1, 32)
    a = np.abs(v)
    bad = ~np.isfinite(v).all(-1)
    with np.errstate(all="ignore"):
        first = np.argmax(a, -1)
        big = np.take_along_axis(v, first[..., None], -1)[..., 0]
        other = np.where((v > 0) != (big > 0)[..., None], a, 0).max(-1)
        step = np.minimum(np.maximum(np.abs(big) / np.float32(8), other / np.float32(7)), np.float32(65504))
        d = np.where(big > 0, -step, step).astype(np.float16)
        d[bad] = np.nan
        d64 = d.astype(np.float64)[..., None]
        code = np.where((d64 == 0) | bad[..., None], 0, np.clip(np.rint(v.astype(np.float64) / d64), -8, 7))
        val = code * d64
    return val.reshape(x.shape), code.reshape(x.shape), d


class Pool:
    """A cache with a shuffled page table, the batch's device arrays, and the values it holds (numpy, per sequence)."""

    def __init__(self, gpu, t, KV, hd, lens, layers=1, layer=0, seed=0, extra_ld=1, pages=None, scale=1.0):
        self.mb, self.t, self.KV, self.hd, self.layer = gpu, t, KV, hd, layer
        rng = np.random.default_rng(seed)
        need = [(L + 63) // 64 for L in lens]
        self.ld = max(need + [1]) + extra_ld
        self.pages = pages or sum(need) + 3
        self.kv = gpu.Kv4(layers, KV, hd, self.pages)
        perm = rng.permutation(self.pages)
        self.table = np.full((len(lens), self.ld), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = perm[at:at + n]; at += n
        self.lens, self.rng = list(lens), rng
        self.k = [(rng.standard_normal((L, KV, hd)) * scale).astype(np.float32) for L in lens]
        self.v = [rng.standard_normal((L, KV, hd)).astype(np.float32) for L in lens]
        self.store()

    def dev(self, a, dtype=np.int32):
        return self.t.from_numpy(np.ascontiguousarray(a, dtype)).cuda()

    def sh(self):
        return self.mb.stream_handle(self.t.cuda.current_stream())

    def batch(self, rows, lens=None, table=None, pad=0, max_rows=None, max_len=None):
        lens = self.lens if lens is None else lens
        row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.row0 = row0
        arrs = [self.dev(row0), self.dev(lens), self.dev(self.table if table is None else table)]
        b = self.mb.Kv4Batch(len(lens), int(row0[-1]) + pad, arrs[0].data_ptr(), arrs[1].data_ptr(), arrs[2].data_ptr(), self.ld,
                             max_rows=max(list(rows) + [0]) if max_rows is None else max_rows,
                             max_len=max(list(lens) + [0]) if max_len is None else max_len)
        b.keep = arrs
        return b

    def store(self):
        if not sum(self.lens):
            return
        k, v = (self.dev(np.concatenate([x.reshape(-1, self.KV * self.hd) for x in y]), np.float32) for y in (self.k, self.v))
        b = self.batch(self.lens)
        self.kv.append_dev(self.layer, k.data_ptr(), v.data_ptr(), b, stream=self.sh())
        self.t.cuda.synchronize()

    def status(self):
        self.mb._ck(self.mb.lib().moty_cuda_kernel_status(0, C.c_void_p(self.sh())))

    def attend(self, q, H, rows, window=0, scale=0.0, **kw):
        b = self.batch(rows, **kw)
        qd = self.dev(q, np.float32)
        ctx = self.t.full((b.c.rows, H * self.hd), 7.0, device="cuda")
        self.kv.attend_dev(self.layer, ctx.data_ptr(), qd.data_ptr(), H, b, window=window, scale=scale, stream=self.sh())
        self.t.cuda.synchronize()
        return ctx.cpu().numpy()


def attend64(k, v, q, pos, G, window=0, scale=None, hidden=None):
    """k, v [T][KV][hd] values held (f64), q [n][H][hd], pos [n] -> (ctx [n][H][hd], tolerance [n][H])"""
    T, KV, hd = k.shape
    scale = 1 / math.sqrt(hd) if scale is None else scale
    ctx, tol = np.zeros(q.shape), np.zeros(q.shape[:2])
    for i, p in enumerate(pos):
        lo = max(0, p - window + 1) if window else 0
        see = np.arange(lo, p + 1)
        if hidden is not None:
            see = see[~hidden[see]]
        if not see.size:
            continue
        for h in range(q.shape[1]):
            kk, vv, qq = k[see, h // G], v[see, h // G], q[i, h].astype(np.float64)
            with np.errstate(all="ignore"):
                s = scale * (kk @ qq)
                A = np.max(scale * (np.abs(kk) @ np.abs(qq)))
                w = np.exp(s - np.max(s))
                ctx[i, h] = (w @ vv) / w.sum()
                ds = (2 * E + 2 * E * (hd / 16 + 16) + 4 * E) * A
                tol[i, h] = np.max(np.abs(vv)) * (2 * ds + 8 * E + 4 * E * (see.size / 16 + 64))
    return ctx, tol


def check(got, want, tol):
    got = got.reshape(want.shape).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    err = np.nan_to_num(np.abs(got - want))
    worst = np.max(err / np.maximum(np.nan_to_num(tol), 1e-30)[..., None]) if err.size else 0
    assert (err <= np.nan_to_num(tol)[..., None]).all(), f"worst error / tolerance {worst:.3g}"


# ---- store and fetch ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("KV,rows,lens", [(1, [1], [1]), (3, [1, 5, 64, 2], [65, 5, 200, 128]), (8, [130], [130])])
def test_append_and_fetch(gpu, t, hd, KV, rows, lens):
    p = Pool(gpu, t, KV, hd, lens, layers=3, layer=1, seed=hd)
    b = p.batch(rows)
    n = sum(rows)
    k = t.full((n, KV * hd), 9.0, device="cuda"); v = k.clone()
    p.kv.fetch_dev(1, k.data_ptr(), v.data_ptr(), b, stream=p.sh())
    want = [np.concatenate([quant(x[L - r:])[0].reshape(-1, KV * hd) for x, L, r in zip(y, lens, rows)]) for y in (p.k, p.v)]
    assert np.array_equal(k.cpu().numpy(), want[0].astype(np.float32)) and np.array_equal(v.cpu().numpy(), want[1].astype(np.float32))
    # the other layers were not touched (the library's memory starts as zero rows)
    for layer in (0, 2):
        p.kv.fetch_dev(layer, k.data_ptr(), v.data_ptr(), b, stream=p.sh())
        assert not k.any() and not v.any()
    p.status()


@pytest.mark.parametrize("nseq", [16, 17, 40, 300])
def test_append_and_fetch_many_sequences(gpu, t, nseq):
    """Rows of many sequences in one batch, some with none."""
    rng = np.random.default_rng(nseq)
    lens = [int(x) for x in rng.integers(1, 90, nseq)]
    p = Pool(gpu, t, 2, 64, lens, seed=nseq)
    rows = [int(min(L, r)) for L, r in zip(lens, rng.choice([0, 0, 1, 1, 3, 20, 90], nseq))]
    n = sum(rows)
    k = t.full((n, 2 * 64), 7.0, device="cuda"); v = k.clone()
    p.kv.fetch_dev(0, k.data_ptr(), v.data_ptr(), p.batch(rows), stream=p.sh())
    for got, held in ((k, p.k), (v, p.v)):
        want = np.concatenate([quant(x[L - r:])[0] for x, L, r in zip(held, lens, rows) if r]).reshape(n, -1)
        assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))
    p.status()


def test_append_strides_and_single_positions(gpu, t):
    """Rows inside wider rows; positions stored one call at a time leave their neighbours as they were."""
    KV, hd, L = 2, 96, 70
    p = Pool(gpu, t, KV, hd, [L, 3], seed=3)
    new_k, new_v = (p.rng.standard_normal((L, KV, hd)).astype(np.float32) for _ in range(2))
    wide = t.zeros((L, 700), device="cuda")
    wide[:, 4:4 + KV * hd] = p.dev(new_k.reshape(L, -1), np.float32)
    wide[:, 300:300 + KV * hd] = p.dev(new_v.reshape(L, -1), np.float32)
    order = p.rng.permutation(L)
    for i, pos in enumerate(order):
        b = p.batch([1, 0], lens=[int(pos) + 1, 3])
        p.kv.append_dev(0, wide.data_ptr() + 4 * (700 * int(pos) + 4), wide.data_ptr() + 4 * (700 * int(pos) + 300), b, stream=p.sh(), ld=700)
        if i in (0, 20, L - 1):
            k = t.empty((L + 3, KV * hd), device="cuda"); v = t.empty_like(k)
            ball = p.batch([L, 3])
            p.kv.fetch_dev(0, k.data_ptr(), v.data_ptr(), ball, stream=p.sh())
            done = np.isin(np.arange(L), order[:i + 1])[:, None, None]
            wk, wv = np.where(done, new_k, p.k[0]), np.where(done, new_v, p.v[0])
            assert np.array_equal(k[:L].cpu().numpy().reshape(wk.shape), quant(wk)[0].astype(np.float32))
            assert np.array_equal(v[:L].cpu().numpy().reshape(wv.shape), quant(wv)[0].astype(np.float32))
            assert np.array_equal(k[L:].cpu().numpy().reshape(p.k[1].shape), quant(p.k[1])[0].astype(np.float32))
    p.status()


def test_append_hard_values(gpu, t):
    """Zeros, signs on a tie, steps that round to nothing, that saturate, ties of the quotient, infinities and NaN."""
    hd = 64
    x = np.random.default_rng(0).standard_normal((64, 1, hd)).astype(np.float32)
    x[0] = 0; x[1] = -0.0; x[2, 0, 0], x[2, 0, 5] = 40, -40; x[3, 0, 5], x[3, 0, 0] = 40, -40
    x[4] *= 1e-7; x[5] *= 1e-8; x[6] *= 3e-5; x[7] *= 1e6; x[8] *= 1e30; x[9, 0, 3] = np.inf; x[10, 0, 40] = -np.inf; x[11, 0, 31] = np.nan
    x[12, 0, :32] = np.arange(-16, 16) / 4; x[13, 0, :32] = np.arange(32) / 8; x[14] = np.float32(1e-45); x[15] = np.finfo(np.float32).max
    x[16, 0, :32] = 8; x[16, 0, 1:17] = np.arange(16) + 0.5 - 8; x[17, 0, :32] = -8; x[17, 0, 1:17] = np.arange(16) + 0.5 - 8
    p = Pool(gpu, t, 1, hd, [64])
    p.k[0], p.v[0] = x, x[::-1].copy()
    p.store()
    k = t.empty((64, hd), device="cuda"); v = t.empty_like(k)
    p.kv.fetch_dev(0, k.data_ptr(), v.data_ptr(), p.batch([64]), stream=p.sh())
    for got, src in ((k, p.k[0]), (v, p.v[0])):
        assert np.array_equal(got.cpu().numpy(), quant(src)[0].astype(np.float32).reshape(64, hd), equal_nan=True)


def test_rows_behind_the_last_sequence_stay(gpu, t):
    KV, hd, H = 2, 64, 4
    p = Pool(gpu, t, KV, hd, [40, 70, 9], seed=5)
    rows, pad = [2, 0, 3], 4
    n = sum(rows)
    q = p.rng.standard_normal((n + pad, H, hd)).astype(np.float32); q[n:] = np.nan
    out = p.attend(q, H, rows, pad=pad)
    assert (out[n:] == 7.0).all() and np.isfinite(out[:n]).all() and (out[:n] != 7.0).any()
    k = t.full((n + pad, KV * hd), 5.0, device="cuda"); v = k.clone()
    b = p.batch(rows, pad=pad)
    p.kv.fetch_dev(0, k.data_ptr(), v.data_ptr(), b, stream=p.sh())
    assert (k[n:] == 5).all() and (v[n:] == 5).all()
    # and an append with NaN in the padding changes no page
    k[n:] = math.nan; v[n:] = math.nan
    p.kv.append_dev(0, k.data_ptr(), v.data_ptr(), b, stream=p.sh())
    again = p.attend(q, H, rows, pad=pad)
    assert np.isfinite(again[:n]).all()
    p.status()


# ---- attention ---------------------------------------------------------------------------------------------------------
CASES = [
    # H, KV, hd, rows, lens, window
    (1, 1, 32, [1], [1], 0),
    (2, 1, 64, [1], [2], 0),
    (16, 8, 128, [1], [1000], 0),
    (8, 2, 128, [1, 1, 1, 1, 1], [1, 64, 65, 129, 700], 0),
    (32, 4, 128, [1, 1], [333, 64], 0),
    (6, 2, 96, [1, 1, 1], [15, 16, 17], 0),
    (5, 1, 160, [1, 2], [300, 77], 0),
    (7, 1, 224, [1, 1], [129, 1], 0),
    (16, 8, 256, [1, 1], [1500, 200], 1024),
    (4, 4, 192, [1, 1], [100, 1000], 7),
    (16, 1, 64, [1, 1], [600, 31], 0),
    (34, 2, 64, [1], [130], 0),
    (4, 2, 64, [4, 1, 3], [4, 50, 600], 0),
    (8, 2, 128, [5, 2], [70, 2], 3),
    (16, 4, 64, [1, 1], [5000, 4097], 0),
    (8, 8, 128, [33], [33], 0),
    (20, 4, 96, [70, 1, 130, 17], [70, 300, 200, 400], 0),
    (16, 8, 256, [65], [190], 0),
    (4, 1, 32, [300], [300], 100),
    (12, 4, 128, [129, 64], [1000, 64], 333),
    (3, 3, 224, [20], [90], 1),
    (64, 4, 64, [9], [200], 0),
    (10, 2, 160, [50, 1], [60, 90], 0),
    (24, 3, 192, [40], [333], 0),
]


@pytest.mark.parametrize("H,KV,hd,rows,lens,window", CASES)
def test_attend(gpu, t, H, KV, hd, rows, lens, window):
    p = Pool(gpu, t, KV, hd, lens, seed=H * hd + len(lens), scale=2.0)
    n = sum(rows)
    q = p.rng.standard_normal((n, H, hd)).astype(np.float32)
    got = p.attend(q, H, rows, window=window)
    again = p.attend(q, H, rows, window=window)
    assert got.tobytes() == again.tobytes()                  # the same bits every time
    at = 0
    for s, (r, L) in enumerate(zip(rows, lens)):
        want, tol = attend64(quant(p.k[s])[0], quant(p.v[s])[0], q[at:at + r], np.arange(L - r, L), H // KV, window)
        check(got[at:at + r], want, tol)
        at += r
    p.status()


@pytest.mark.parametrize("scale", [0.02, 1.0, 5.0])
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_peaked_and_flat(gpu, t, scale, rows):
    """Scores of thousands (one position takes all), scores of nothing, rows of very different size, one huge value row."""
    H, KV, hd, L = 4, 2, 64, 333
    p = Pool(gpu, t, KV, hd, [L], seed=1, scale=8.0)
    p.k[0][::7] *= 1e-3; p.v[0][5] *= 3000.0; p.v[0][100:] *= 1e-3; p.v[0][L - rows - 1, :, :32] *= 1e4
    p.store()
    q = p.rng.standard_normal((rows, H, hd)).astype(np.float32)
    q[:, 1] *= 50; q[:, 2] *= 1e-6; q[:, 3] = 0
    got = p.attend(q, H, [rows], scale=scale)
    want, tol = attend64(quant(p.k[0])[0], quant(p.v[0])[0], q, np.arange(L - rows, L), H // KV, scale=scale)
    check(got, want, tol)


@pytest.mark.parametrize("mag", [1e-30, 1e-12, 1e12, 1e30])
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_query_range(gpu, t, mag, rows):
    """Query rows far from 1, brought back by the scale."""
    H, KV, hd, L = 4, 2, 64, 90
    p = Pool(gpu, t, KV, hd, [L], seed=2)
    q = (p.rng.standard_normal((rows, H, hd)) * mag).astype(np.float32)
    sc = np.float32(0.3 / mag)
    got = p.attend(q, H, [rows], scale=float(sc))
    want, tol = attend64(quant(p.k[0])[0], quant(p.v[0])[0], q, np.arange(L - rows, L), H // KV, scale=float(sc))
    check(got, want, tol)


@pytest.mark.parametrize("rows", [1, 3, 50])
def test_attend_absent_pages_and_what_lies_behind_the_mask(gpu, t, rows):
    """Pages freed in front of the window; pages absent inside it; a row that sees nothing; NaN in positions past a row's own
    and in freed pages never reach a result, NaN in a seen value does."""
    H, KV, hd, L = 8, 2, 128, 400
    p = Pool(gpu, t, KV, hd, [L, 200], seed=4)
    p.k[0][64:128] = np.nan; p.v[0][64:128] = np.inf                     # page 1 of sequence 0 will be absent
    p.v[1][150, 0, 40] = np.nan                                          # seen by KV head 0's queries of sequence 1, dims 32..63
    p.store()
    table = p.table.copy(); table[0, 1] = -1; table[0, 3] = -1
    hidden = np.zeros(L, bool); hidden[64:128] = True; hidden[192:256] = True
    q = p.rng.standard_normal((rows + 1, H, hd)).astype(np.float32)
    got = p.attend(q, H, [rows, 1], table=table)
    want, tol = attend64(np.nan_to_num(quant(p.k[0])[0]), np.nan_to_num(quant(p.v[0])[0]), q[:rows], np.arange(L - rows, L), H // KV, hidden=hidden)
    check(got[:rows], want, tol)
    out1 = got[rows].reshape(H, hd)
    assert np.isnan(out1[:4, 32:64]).all() and np.isfinite(np.delete(out1[:4], np.arange(32, 64), axis=1)).all() and np.isfinite(out1[4:]).all()
    # lengths that end in front of stored rows: what lies behind is not seen (rows 30.. of sequence 0 hold numbers, later pages NaN)
    lens = [60, 140]
    p.v[0][60:64] = np.nan; p.k[0][60:64] = np.inf
    p.store()
    r = min(rows, 60)
    got = p.attend(q[:r + 1], H, [r, 1], lens=lens, table=table)
    want, tol = attend64(quant(p.k[0][:60])[0], quant(p.v[0][:60])[0], q[:r], np.arange(60 - r, 60), H // KV)
    check(got[:r], want, tol)
    # a window that lies wholly in an absent page: nothing to see
    got = p.attend(q[:2], H, [1, 1], lens=[100, 140], table=table, window=30)
    assert (got[0] == 0).all() and np.isfinite(got[1]).all() and (got[1] != 0).any()
    p.status()
    got = p.attend(q[:1], H, [1, 0], table=np.full_like(p.table, -1))
    assert (got == 0).all()
    p.status()


@pytest.mark.parametrize("rows", [1, 40])
def test_attend_query_that_is_not_finite(gpu, t, rows):
    """An infinity or NaN in a query row makes that row of that head NaN and no other."""
    H, KV, hd, L = 4, 2, 64, 70
    p = Pool(gpu, t, KV, hd, [L], seed=6)
    q = p.rng.standard_normal((rows, H, hd)).astype(np.float32)
    clean = p.attend(q, H, [rows]).reshape(rows, H, hd)
    q[0, 1, 3] = np.nan; q[rows - 1, 2, 60] = np.inf
    got = p.attend(q, H, [rows]).reshape(rows, H, hd)
    hit = np.zeros((rows, H), bool); hit[0, 1] = True; hit[rows - 1, 2] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


def test_attend_strided_queries_and_another_stream(gpu, t):
    H, KV, hd = 6, 2, 96
    p = Pool(gpu, t, KV, hd, [100, 30], seed=7)
    q = p.rng.standard_normal((2, H, hd)).astype(np.float32)
    plain = p.attend(q, H, [1, 1])
    wide = t.zeros((2, 1000), device="cuda"); wide[:, 8:8 + H * hd] = p.dev(q.reshape(2, -1), np.float32)
    t.cuda.synchronize()
    st = t.cuda.Stream()
    with t.cuda.stream(st):
        b = p.batch([1, 1])
        ctx = t.empty((2, H * hd), device="cuda")
        p.kv.attend_dev(0, ctx.data_ptr(), wide.data_ptr() + 32, H, b, stream=gpu.stream_handle(st), q_ld=1000)
    st.synchronize()
    assert ctx.cpu().numpy().tobytes() == plain.tobytes()
    # and the library's own stream (NULL)
    ctx.zero_(); t.cuda.synchronize()
    p.kv.attend_dev(0, ctx.data_ptr(), wide.data_ptr() + 32, H, b, q_ld=1000)
    gpu.sync(0)
    assert ctx.cpu().numpy().tobytes() == plain.tobytes()

# A table with room for much longer sequences than there are: the cut of the work follows the limits, so that the same small
# batch also runs through the kernels and the many short spans of large ones.
ROOM = [0, 150]


@pytest.mark.parametrize("H,KV,hd,rows,lens,window", [c for c in CASES if max(c[3]) > 1])
def test_attend_with_room(gpu, t, H, KV, hd, rows, lens, window):
    p = Pool(gpu, t, KV, hd, lens, seed=H * hd + len(lens), scale=2.0, extra_ld=500)
    q = p.rng.standard_normal((sum(rows), H, hd)).astype(np.float32)
    got = p.attend(q, H, rows, window=window, max_len=p.ld * 64)
    assert got.tobytes() == p.attend(q, H, rows, window=window, max_len=p.ld * 64).tobytes()
    at = 0
    for s, (r, L) in enumerate(zip(rows, lens)):
        want, tol = attend64(quant(p.k[s])[0], quant(p.v[s])[0], q[at:at + r], np.arange(L - r, L), H // KV, window)
        check(got[at:at + r], want, tol)
        at += r
    p.status()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("rows", [1, 3, 20, 70])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
def test_attend_values_and_keys_that_are_not_finite(gpu, t, hd, rows, room):
    """A NaN value reaches the rows that see its position, in its group's 32 dims, however small its weight; an infinite key
    makes the rows that see it NaN altogether; no other row or head changes."""
    H, KV, L, G = 8, 2, 300, 4
    p = Pool(gpu, t, KV, hd, [L], seed=hd + rows, scale=2.0, extra_ld=1 + room)
    q = p.rng.standard_normal((rows, H, hd)).astype(np.float32)
    pos, scale = np.arange(L - rows, L), 4.0                 # (weights from 1 down to what underflows)
    clean = p.v[0].copy()
    g = hd // 64                                             # a group of 32 dims
    # one that all see, one that half of the rows see, in different heads
    at = [(70, 0), (L - 1 - rows // 2, 1)]
    for w, h in at:
        p.v[0][w, h, 32 * g + 5] = np.nan
    p.store()
    got = p.attend(q, H, [rows], scale=scale, max_len=p.ld * 64).reshape(rows, H, hd)
    ql = clean.copy()
    for w, h in at:
        ql[w, h, 32 * g:32 * g + 32] = 0
    want, tol = attend64(quant(p.k[0])[0], quant(ql)[0], q, pos, G, scale=scale)
    for w, h in at:
        want[pos >= w, h * G:(h + 1) * G, 32 * g:32 * g + 32] = np.nan
    check(got, want, tol)
    # keys
    p.v[0] = clean
    for w, h in at:
        p.k[0][w, h, 3] = np.inf
    p.store()
    got = p.attend(q, H, [rows], scale=scale, max_len=p.ld * 64).reshape(rows, H, hd)
    kl = np.where(np.isfinite(p.k[0]), p.k[0], 0)
    want, tol = attend64(quant(kl)[0], quant(clean)[0], q, pos, G, scale=scale)
    for w, h in at:
        want[pos >= w, h * G:(h + 1) * G] = np.nan
    check(got, want, tol)
    p.status()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kmag,vmag", [(3e4, 1.0), (1.0, 9e4), (1e-6, 1e-6), (3e4, 9e4)])
def test_attend_step_range(gpu, t, hd, rows, kmag, vmag, room):
    """Steps from the smallest f16 numbers to nearly the largest."""
    H, KV, L = 8, 2, 200
    p = Pool(gpu, t, KV, hd, [L], seed=hd + rows, scale=kmag, extra_ld=1 + room)
    p.v[0] *= np.float32(vmag)
    p.store()
    q = p.rng.standard_normal((rows, H, hd)).astype(np.float32)
    scale = float(np.float32(1 / (kmag * math.sqrt(hd))))
    got = p.attend(q, H, [rows], scale=scale, max_len=p.ld * 64)
    want, tol = attend64(quant(p.k[0])[0], quant(p.v[0])[0], q, np.arange(L - rows, L), H // KV, scale=scale)
    check(got, want, tol)
    p.status()


@pytest.mark.parametrize("nseq,rows,H,KV,hd,L", [(5, 40, 128, 16, 64, 33285), (90, 1, 16, 8, 32, 17001), (3, 20, 64, 32, 160, 9000)])
def test_attend_one_long_sequence_among_short_ones(gpu, t, nseq, rows, H, KV, hd, L):
    """More units than the GPU holds CTAs, and more pages in one sequence than a CTA's list of pages has room for."""
    lens = [rows + 3 * s for s in range(nseq)]
    lens[1] = L
    p = Pool(gpu, t, KV, hd, lens, seed=7)
    q = p.rng.standard_normal((nseq * rows, H, hd)).astype(np.float32)
    got = p.attend(q, H, [rows] * nseq).reshape(-1, H, hd)
    for s in (0, 1, 2, nseq - 1):
        k, v = quant(p.k[s])[0], quant(p.v[s])[0]
        for i, h in ((0, 0), (rows - 1, H - 1), (rows // 2, H // 2)):
            g, row = h // (H // KV), s * rows + i
            want, tol = attend64(k[:, g:g + 1], v[:, g:g + 1], q[row:row + 1, h:h + 1], np.array([lens[s] - rows + i]), 1)
            check(got[row:row + 1, h:h + 1], want, tol)
    p.status()


@pytest.mark.parametrize("H,KV,nseq", [(128, 16, 7), (64, 16, 8), (16, 16, 40)])
def test_attend_long_sums_of_one_sign(gpu, t, H, KV, nseq):
    """Flat weights and positive values: all sums grow evenly.  The matrix unit cuts each of its sums off by at most 2^-23 of the
    sum so far.  Of at most 20 pages of two products, 16 where sums are passed on, or 32 of one, that is 20 x 2^-23 of the
    whole at most and half of that on the average; passing on (31 times at most), four warps, the spans (fewer than 32) and
    the quotient round to nearest, half a 2^-23 each at most, the earlier ones of smaller sums: another 20 x 2^-23 at most
    and nothing on the average.  A score (below 2 in magnitude) is off by less than 2 x 2^-23 x 8, its weight by that much
    and the exponential's 2 x 2^-23: another 20."""
    hd, L = 32, 31680
    p = Pool(gpu, t, KV, hd, [L], seed=H)
    p.v[0] = np.abs(p.v[0]) + np.float32(0.5)
    p.store()
    q = p.rng.standard_normal((nseq, H, hd)).astype(np.float32)
    got = p.attend(q, H, [1] * nseq, lens=[L] * nseq, table=np.repeat(p.table, nseq, 0), scale=0.05).reshape(nseq, H, hd)
    k, v = quant(p.k[0])[0], quant(p.v[0])[0]
    rel = []
    for s, h in [(0, 0), (0, H - 1), (nseq - 1, H // 2), (nseq // 2, 1)]:
        want, _ = attend64(k[:, h // (H // KV)][:, None], v[:, h // (H // KV)][:, None], q[s:s + 1, h:h + 1], np.array([L - 1]), 1, scale=0.05)
        rel.append((got[s, h] - want[0, 0]) / want[0, 0])
    rel = np.array(rel)
    assert np.max(np.abs(rel)) <= 60 * 2.0**-23
    assert abs(np.mean(rel)) <= 10 * 2.0**-23
    p.status()


@pytest.mark.parametrize("rows", [1, 20])
def test_attend_does_not_depend_on_the_neighbours(gpu, t, rows):
    """A sequence's result is the same bits alone with the same limits and beside others."""
    H, KV, hd = 8, 2, 128
    p = Pool(gpu, t, KV, hd, [900, 77, 300], seed=8)
    q = p.rng.standard_normal((3 * rows, H, hd)).astype(np.float32)
    both = p.attend(q, H, [rows] * 3)
    for s in range(3):
        r = [0, 0, 0]; r[s] = rows
        one = p.attend(q[s * rows:(s + 1) * rows], H, r, max_rows=rows)
        assert one.tobytes() == both[s * rows:(s + 1) * rows].tobytes()


def test_offsets_past_32_bits(gpu, t):
    """Units that begin beyond 4 GiB of the pool."""
    layers, KV, hd, H = 64, 16, 256, 16
    pages = (5 << 30) // gpu.Kv4.page_bytes(layers, KV, hd) + 2
    p = Pool(gpu, t, KV, hd, [100, 70], layers=layers, layer=63, seed=9, pages=pages)
    p.table[:, :2] = [[pages - 1, 1], [0, pages - 2]]
    p.store()
    q = p.rng.standard_normal((2, H, hd)).astype(np.float32)
    got = p.attend(q, H, [1, 1])
    for s, L in enumerate(p.lens):
        want, tol = attend64(quant(p.k[s])[0], quant(p.v[s])[0], q[s:s + 1], [L - 1], 1)
        check(got[s:s + 1], want, tol)
    new = t.tensor([pages - 3], device="cuda", dtype=t.int32)
    src, dst = t.tensor([0], device="cuda", dtype=t.int32), t.tensor([1], device="cuda", dtype=t.int32)
    tab, ln = p.dev(p.table), p.dev(p.lens)
    p.kv.fork_dev(1, src.data_ptr(), dst.data_ptr(), new.data_ptr(), 2, ln.data_ptr(), tab.data_ptr(), p.ld, stream=p.sh())
    p.table = tab.cpu().numpy()
    assert p.table[1, :2].tolist() == [pages - 1, pages - 3]
    again = p.attend(q[[0, 0]], H, [1, 1], lens=[100, 100])
    assert again[0].tobytes() == again[1].tobytes() == got[0].tobytes()
    p.status()
    p.kv.close()


# ---- arguments and batches that are refused ------------------------------------------------------------------------------
def test_refused_arguments(gpu, t):
    p = Pool(gpu, t, 2, 64, [10])
    x = t.zeros((1, 4096), device="cuda")
    ok = p.batch([1])
    a = x.data_ptr()
    mk = lambda **kw: gpu.Kv4Batch(**{**dict(nseq=1, rows=1, row0_ptr=ok.c.row0_dev, len_ptr=ok.c.len_dev, table_ptr=ok.c.table_dev, table_ld=p.ld,
                                             max_rows=1, max_len=10), **kw})
    bad = [
        lambda: p.kv.append_dev(1, a, a, ok), lambda: p.kv.append_dev(-1, a, a, ok), lambda: p.kv.append_dev(0, 0, a, ok),
        lambda: p.kv.append_dev(0, a, a + 4, ok), lambda: p.kv.append_dev(0, a, a, ok, ld=127), lambda: p.kv.append_dev(0, a, a, ok, ld=130),
        lambda: p.kv.append_dev(0, a, a, mk(nseq=-1)), lambda: p.kv.append_dev(0, a, a, mk(rows=-1)), lambda: p.kv.append_dev(0, a, a, mk(table_ld=0)),
        lambda: p.kv.append_dev(0, a, a, mk(row0_ptr=0)), lambda: p.kv.append_dev(0, a, a, mk(len_ptr=0)), lambda: p.kv.append_dev(0, a, a, mk(table_ptr=0)),
        lambda: p.kv.fetch_dev(0, a, 0, ok), lambda: p.kv.fetch_dev(0, a + 8, a, ok),
        lambda: p.kv.attend_dev(0, a, a, 3, ok), lambda: p.kv.attend_dev(0, a, a, 0, ok), lambda: p.kv.attend_dev(0, a, a, 4, ok, window=-1),
        lambda: p.kv.attend_dev(0, a, a, 4, ok, scale=-1.0), lambda: p.kv.attend_dev(0, a, a, 4, ok, scale=math.nan),
        lambda: p.kv.attend_dev(0, a, a, 4, ok, scale=math.inf), lambda: p.kv.attend_dev(0, a, a, 4, ok, q_ld=200),
        lambda: p.kv.attend_dev(0, a, a, 4, mk(max_rows=2)), lambda: p.kv.attend_dev(0, a, a, 4, mk(max_len=64 * p.ld + 1)),
        lambda: p.kv.attend_dev(0, a, 0, 4, ok), lambda: p.kv.attend_dev(0, a + 4, a, 4, ok),
        lambda: p.kv.append_rope_dev(0, 4, a, a, a, ok, 63, 1e4, 1e-6), lambda: p.kv.append_rope_dev(0, 4, a, a, a, ok, 66, 1e4, 1e-6),
        lambda: p.kv.append_rope_dev(0, 4, a, a, a, ok, 33, 1e4, 1e-6, gemma=True), lambda: p.kv.append_rope_dev(0, 4, a, a, a, ok, 64, 0.0, 1e-6),
        lambda: p.kv.append_rope_dev(0, 4, 0, a, a, ok, 64, 1e4, 1e-6), lambda: p.kv.append_rope_dev(0, -1, a, a, a, ok, 64, 1e4, 1e-6),
        lambda: p.kv.fork_dev(-1, a, a, a, 1, a, a, 1), lambda: p.kv.fork_dev(1, 0, a, a, 1, a, a, 1), lambda: p.kv.fork_dev(1, a, a, a, 1, a, a, 0),
        lambda: p.kv.compact_dev(-1, a, a, 0, 0, 0), lambda: p.kv.compact_dev(1, a, 0, 0, 0, 0), lambda: p.kv.compact_dev(0, 0, 0, 4, a, 0),
        lambda: p.kv.compact_dev(p.pages + 1, a, a, 0, 0, 0),
        lambda: gpu.Kv4(1, 2, 64, 4, mem_ptr=t.zeros(64).pin_memory().data_ptr() // 128 * 128),
        lambda: gpu.Kv4(1, 2, 64, 4, device=9),
        lambda: p.kv.alloc(p.pages + 1), lambda: p.kv.alloc(-1), lambda: p.kv.release([0]), lambda: p.kv.retain([p.pages]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(gpu.MotyCudaError):
            f()
            pytest.fail(f"call {i} was accepted")
    # empty calls do nothing
    p.kv.append_dev(0, a, a, mk(nseq=0)); p.kv.append_dev(0, a, a, mk(rows=0)); p.kv.attend_dev(0, a, a, 4, mk(nseq=0))
    p.kv.attend_dev(0, a, a, 4, mk(rows=0, max_rows=0)); p.kv.fork_dev(0, a, a, a, 1, a, a, 1); p.kv.compact_dev(0, 0, 0, 0, 0, 0)
    t.cuda.synchronize()
    p.status()


def test_attend_of_more_pairs_than_it_counts_is_refused(gpu, t):
    p = Pool(gpu, t, 2, 64, [10])
    a, ok = t.zeros(4096, device="cuda").data_ptr(), p.batch([1])
    for rows, H in ((1 << 29, 4), (1 << 20, 2048), (0x7fffffff, 2)):
        b = gpu.Kv4Batch(1, rows, ok.c.row0_dev, ok.c.len_dev, ok.c.table_dev, p.ld, max_rows=1, max_len=10)
        with pytest.raises(gpu.MotyCudaError):
            p.kv.attend_dev(0, a, a, H, b)


def test_attend_of_a_length_past_2_30_is_refused(gpu, t):
    p = Pool(gpu, t, 2, 64, [10])
    a, ok = t.zeros(4096, device="cuda").data_ptr(), p.batch([1])
    mk = lambda **kw: gpu.Kv4Batch(1, 1, ok.c.row0_dev, ok.c.len_dev, ok.c.table_dev, 1 << 25, max_rows=1, **kw)
    for n in ((1 << 30) + 1, 0x7fffffff):
        with pytest.raises(gpu.MotyCudaError):
            p.kv.attend_dev(0, a, a, 4, mk(max_len=n))
    assert mk().c.max_len == 1 << 30                        # what the binding gives a table of that width


@pytest.mark.parametrize("what", ["len_past_table", "len_past_max", "rows_more_than_len", "row0_negative", "row0_past_rows", "row0_back",
                                  "rows_past_max", "page_past_pool", "page_negative"])
@pytest.mark.parametrize("big", [False, True])
def test_batches_that_are_none(gpu, t, what, big):
    """Arrays that do not describe a batch: nothing is touched that is not the batch's, the sound sequence keeps its result,
    and the status reports it once.  (Every access is bounded by the index functions that the CPU tests check.)"""
    H, KV, hd = 4, 2, 64
    r = 40 if big else 1
    p = Pool(gpu, t, KV, hd, [100, 130], seed=11, pages=8)
    row0, lens, table = np.array([0, r, 2 * r], np.int32), np.array([100, 130], np.int32), p.table.copy()
    max_rows, max_len = r, 130
    if what == "len_past_table": lens[1] = 64 * p.ld + 1
    if what == "len_past_max": max_len = 129
    if what == "rows_more_than_len": lens[1] = r - 1
    if what == "row0_negative": row0[0] = -3
    if what == "row0_past_rows": row0[2] = 2 * r + 1
    if what == "row0_back": row0[2] = r - 1
    if what == "rows_past_max": max_rows = r - 1
    if what == "page_past_pool": table[1, 1] = p.pages
    if what == "page_negative": table[1, 1] = -7
    q = p.rng.standard_normal((2 * r, H, hd)).astype(np.float32)
    good = p.attend(q, H, [r, r])
    arrs = [p.dev(row0), p.dev(lens), p.dev(table)]
    b = gpu.Kv4Batch(2, 2 * r, *(x.data_ptr() for x in arrs), p.ld, max_rows=max_rows, max_len=max_len)
    qd = p.dev(q, np.float32)
    ctx = t.full((2 * r + 2, H * hd), 7.0, device="cuda")
    p.kv.attend_dev(0, ctx.data_ptr() + 4 * H * hd, qd.data_ptr(), H, b, stream=p.sh())
    t.cuda.synchronize()
    out = ctx.cpu().numpy()
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    if what in ("rows_past_max", "row0_negative"):
        pass                                                  # (the first sequence is affected too)
    else:
        check(out[1:1 + r], good[:r].reshape(r, H, hd).astype(np.float64), np.full((r, H), 1e-5))
    with pytest.raises(gpu.MotyCudaError, match="4-bit KV"):
        p.status()
    p.status()                                                # reported once
    # stores and fetches of the same arrays: the first sequence's rows or nothing
    if what not in ("len_past_max", "rows_past_max"):
        k = t.zeros((2 * r, KV * hd), device="cuda")
        p.kv.fetch_dev(0, k.data_ptr(), k.data_ptr(), b, stream=p.sh())
        kd = t.zeros((2 * r, KV * hd), device="cuda")
        p.kv.append_dev(0, kd.data_ptr(), kd.data_ptr(), b, stream=p.sh())
        t.cuda.synchronize()
        if what.startswith("page") and not big:
            p.status()                                        # (the one row lies at position 129, in the sound third page)
        else:
            with pytest.raises(gpu.MotyCudaError, match="4-bit KV"):
                p.status()


# ---- pages -------------------------------------------------------------------------------------------------------------
def _mem(t, gpu, layers, KV, hd, pages, seed):
    g = t.Generator(device="cuda").manual_seed(seed)
    return t.randint(0, 256, (pages, gpu.Kv4.page_bytes(layers, KV, hd)), generator=g, device="cuda", dtype=t.uint8)


@pytest.mark.parametrize("layers,KV,hd", [(1, 1, 32), (3, 2, 96), (28, 8, 128)])
def test_fork(gpu, t, layers, KV, hd):
    pages, ld = 20, 6
    mem = _mem(t, gpu, layers, KV, hd, pages, 1); before = mem.cpu().numpy()
    kv = gpu.Kv4(layers, KV, hd, pages, mem_ptr=mem.data_ptr())
    table = np.full((7, ld), -1, np.int32)
    table[0, :3] = [4, 9, 2]; table[1, :2] = [7, 0]; table[2, :6] = [11, -1, 12, 13, 14, 15]; table[3:] = 19
    lens = np.array([150, 128, 384, 5, 5, 5, 5], np.int32)
    src, dst, new = [0, 0, 1, 2], [4, 3, 6, 5], [17, 5, -1, -1]
    d = lambda a: t.tensor(a, device="cuda", dtype=t.int32)
    S, D, N, T, L = d(src), d(dst), d(new), d(table), d(lens)
    kv.fork_dev(4, S.data_ptr(), D.data_ptr(), N.data_ptr(), 7, L.data_ptr(), T.data_ptr(), ld, stream=gpu.stream_handle(t.cuda.current_stream()))
    t.cuda.synchronize()
    want = before.copy(); want[17] = before[2]; want[5] = before[2]
    table[4] = [4, 9, 17, -1, -1, -1]; table[3] = [4, 9, 5, -1, -1, -1]; table[6] = [7, 0, -1, -1, -1, -1]; table[5] = table[2]
    assert np.array_equal(mem.cpu().numpy(), want) and np.array_equal(T.cpu().numpy(), table)
    assert L.cpu().tolist() == [150, 128, 384, 150, 150, 384, 128]
    assert gpu.lib().moty_cuda_kernel_status(0, None) == 0


@pytest.mark.parametrize("src,dst,new,sound", [
    ([0, 1], [1, 2], [5, 6], []),               # target 1 is a source; then its fork is refused, and so is ... the other is sound
    ([0, 1], [3, 3], [5, 6], []),               # one target twice
    ([0, 1], [2, 3], [5, 5], []),               # one fresh page twice
    ([0, 9], [2, 3], [5, 6], [0]), ([0, -1], [2, 3], [5, 6], [0]), ([0, 1], [2, 4], [5, 6], [0]), ([0, 1], [2, -1], [5, 6], [0]),
    ([0, 1], [2, 3], [5, 8], [0]), ([0, 1], [2, 3], [5, -1], [0]),
])
def test_forks_that_are_refused(gpu, t, src, dst, new, sound):
    layers, KV, hd, pages, ld = 2, 1, 64, 8, 3
    mem = _mem(t, gpu, layers, KV, hd, pages, 2); before = mem.cpu().numpy()
    kv = gpu.Kv4(layers, KV, hd, pages, mem_ptr=mem.data_ptr())
    table = np.full((4, ld), -1, np.int32); table[0, :2] = [0, 1]; table[1, :2] = [2, 3]
    lens = np.array([70, 100, 0, 0], np.int32)
    d = lambda a: t.tensor(a, device="cuda", dtype=t.int32)
    S, D, N, T, L = d(src), d(dst), d(new), d(table), d(lens)
    kv.fork_dev(2, S.data_ptr(), D.data_ptr(), N.data_ptr(), 4, L.data_ptr(), T.data_ptr(), ld, stream=gpu.stream_handle(t.cuda.current_stream()))
    t.cuda.synchronize()
    assert gpu.lib().moty_cuda_kernel_status(0, gpu.stream_handle(t.cuda.current_stream())) == -6
    want, wl = before.copy(), lens.copy()
    if src == [0, 1] and dst == [1, 2]:          # the fork 1 -> 2 does not depend on the refused one
        sound = [1]
    for f in sound:
        want[new[f]] = before[table[src[f], lens[src[f]] // 64]]
        table[dst[f]] = table[src[f]]; table[dst[f], lens[src[f]] // 64] = new[f]; wl[dst[f]] = lens[src[f]]
    assert np.array_equal(mem.cpu().numpy(), want) and np.array_equal(T.cpu().numpy(), table) and np.array_equal(L.cpu().numpy(), wl)


@pytest.mark.parametrize("layers,KV,hd,pages,seed", [(1, 1, 32, 9, 0), (5, 3, 96, 40, 1), (28, 8, 128, 60, 2), (2, 1, 64, 700, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(gpu, t, layers, KV, hd, pages, seed, in_place):
    mem = _mem(t, gpu, layers, KV, hd, pages, seed); before = mem.cpu().numpy()
    kv = gpu.Kv4(layers, KV, hd, pages, mem_ptr=mem.data_ptr())
    rng = np.random.default_rng(seed)
    ids = kv.alloc(pages)
    gone = rng.choice(pages, pages * 2 // 3, replace=False)
    kv.release(gone)
    live = np.setdiff1d(ids, gone)
    table = np.where(rng.random((13, 17)) < 0.3, -1, rng.choice(live, (13, 17))).astype(np.int32)
    src, dst = kv.compact_plan()
    assert len(src) == np.sum(live >= len(live)) and kv.free_pages() == len(gone)
    d = lambda a: t.tensor(np.asarray(a, np.int32), device="cuda")
    S, D, T = d(src), d(dst), d(table)
    out = T if in_place else t.full_like(T, 99)
    kv.compact_dev(len(src), S.data_ptr(), D.data_ptr(), T.numel(), T.data_ptr(), out.data_ptr(), stream=gpu.stream_handle(t.cuda.current_stream()))
    t.cuda.synchronize()
    ren = {int(a): int(b) for a, b in zip(src, dst)}
    want = before.copy()
    for a, b in ren.items():
        want[b] = before[a]
    assert np.array_equal(mem.cpu().numpy(), want)
    assert np.array_equal(out.cpu().numpy(), np.vectorize(lambda v: ren.get(int(v), int(v)))(table))
    assert gpu.lib().moty_cuda_kernel_status(0, None) == 0
    assert kv.alloc(len(gone)).tolist() == list(range(len(live), pages))       # the books follow


@pytest.mark.parametrize("src,dst", [([5, 4], [0, 1]), ([4, 5], [1, 0]), ([4, 4], [0, 1]), ([4, 5], [1, 1]), ([3, 5], [0, 3]),
                                     ([3, 8], [0, 1]), ([-1, 5], [0, 1]), ([4, 5], [-2, 1])])
def test_compactions_that_are_refused(gpu, t, src, dst):
    """Lists that are not ascending, meet, or leave the pool: reported, and no page that is not a target changes."""
    mem = _mem(t, gpu, 2, 1, 64, 8, 5); before = mem.cpu().numpy()
    kv = gpu.Kv4(2, 1, 64, 8, mem_ptr=mem.data_ptr())
    d = lambda a: t.tensor(a, device="cuda", dtype=t.int32)
    S, D = d(src), d(dst)
    kv.compact_dev(2, S.data_ptr(), D.data_ptr(), 0, 0, 0, stream=gpu.stream_handle(t.cuda.current_stream()))
    t.cuda.synchronize()
    assert gpu.lib().moty_cuda_kernel_status(0, gpu.stream_handle(t.cuda.current_stream())) == -6
    after = mem.cpu().numpy()
    for pg in range(8):
        if pg not in dst:
            assert np.array_equal(after[pg], before[pg])


# ---- norm, rotation, store ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,KV,hd,rot,gemma,gains", [(4, 2, 64, 64, False, True), (8, 8, 128, 128, False, True), (6, 2, 96, 32, False, False),
                                                     (4, 2, 256, 96, True, True), (2, 1, 160, 80, True, True), (2, 2, 128, 0, False, True)])
def test_append_rope_matches_the_attention_core(gpu, t, H, KV, hd, rot, gemma, gains):
    """q and k come out of append_rope with the bits that attn_core_dev leaves, at every row's own position; what is stored is
    the quantised result."""
    rng = np.random.default_rng(hd)
    rows, lens = [3, 1, 5], [3, 77, 130]
    n = sum(rows)
    q, k, v = (rng.standard_normal((n, h * hd)).astype(np.float32) for h in (H, KV, KV))
    g = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if gains else None for _ in range(3)]
    vn = g[2] if gemma else None
    theta, eps = 1e4, 1e-6
    p = Pool(gpu, t, KV, hd, lens, seed=1)
    # the core, one sequence at a time
    wq, wk = [], []
    at = 0
    for r, L in zip(rows, lens):
        a = gpu.Attn(H, KV, hd, L, theta=theta, eps=eps, rot=rot, qn=g[0], kn=g[1], gemma=gemma, vn=vn)
        qd, kd, vd = (p.dev(x[at:at + r], np.float32) for x in (q, k, v))
        ctx = t.empty((r, H * hd), device="cuda")
        a.core_dev(ctx.data_ptr(), qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), r, L - r, stream=p.sh())
        t.cuda.synchronize()
        wq.append(qd.cpu().numpy()); wk.append(kd.cpu().numpy())
        a.close(); at += r
    wq, wk = np.concatenate(wq), np.concatenate(wk)
    wv = v.reshape(n, KV, hd)
    if vn is not None:
        ms = (wv.astype(np.float64) ** 2).mean(-1).astype(np.float32)
        wv = (wv * (np.float32(1) / np.sqrt(ms + np.float32(eps)))[..., None]) * vn
    width = (H + 2 * KV) * hd + 4                                  # one fused row [q | k | v], padded
    buf = t.zeros((n, width), device="cuda")
    for x, off in ((q, 0), (k, H * hd), (v, (H + KV) * hd)):
        buf[:, off:off + x.shape[1]] = p.dev(x, np.float32)
    gd = [0 if x is None else p.dev(x, np.float32) for x in (g[0], g[1], vn)]
    ptr = [x if isinstance(x, int) else x.data_ptr() for x in gd]
    b0 = buf.data_ptr()
    b = p.batch(rows)
    p.kv.append_rope_dev(0, H, b0, b0 + 4 * H * hd, b0 + 4 * (H + KV) * hd, b, rot, theta, eps, *ptr, gemma=gemma, stream=p.sh(), q_ld=width, kv_ld=width)
    t.cuda.synchronize()
    got = buf.cpu().numpy()
    assert got[:, :H * hd].tobytes() == wq.tobytes() and got[:, H * hd:(H + KV) * hd].tobytes() == wk.tobytes()
    assert np.array_equal(got[:, (H + KV) * hd:(H + 2 * KV) * hd], v) and not got[:, -4:].any()
    kh, vh = t.empty((n, KV * hd), device="cuda"), t.empty((n, KV * hd), device="cuda")
    p.kv.fetch_dev(0, kh.data_ptr(), vh.data_ptr(), b, stream=p.sh())
    assert np.array_equal(kh.cpu().numpy(), quant(wk.reshape(n, KV, hd))[0].astype(np.float32).reshape(n, -1))
    assert np.array_equal(vh.cpu().numpy(), quant(wv.astype(np.float32))[0].astype(np.float32).reshape(n, -1))
    p.status()


# ---- graphs ------------------------------------------------------------------------------------------------------------
def test_captured_steps_follow_the_batch_arrays(gpu, t):
    """append + attend captured once, replayed while lengths, table and rows move; an eager call between the replays."""
    H, KV, hd = 8, 2, 128
    p = Pool(gpu, t, KV, hd, [200, 10, 63], seed=12, extra_ld=3, pages=20)
    used = set(p.table[p.table >= 0].tolist()); free = [i for i in range(20) if i not in used]
    st = t.cuda.Stream()
    lens = p.dev(p.lens); table = p.dev(p.table); row0 = p.dev([0, 1, 2, 3])
    q, k, v = (t.zeros((3, h * hd), device="cuda") for h in (H, KV, KV)); ctx = t.zeros((3, H * hd), device="cuda")
    b = gpu.Kv4Batch(3, 3, row0.data_ptr(), lens.data_ptr(), table.data_ptr(), p.ld, max_rows=1, max_len=64 * p.ld)
    t.cuda.synchronize()

    def body():
        sh = gpu.stream_handle(t.cuda.current_stream())
        p.kv.append_dev(0, k.data_ptr(), v.data_ptr(), b, stream=sh)
        p.kv.attend_dev(0, ctx.data_ptr(), q.data_ptr(), H, b, stream=sh)

    with t.cuda.stream(st):
        body()                                                 # (stores zero rows at the last positions: stored again below)
    st.synchronize()
    gpu._ck(gpu.lib().moty_cuda_scratch_freeze(0, 1))
    try:
        p.store(); t.cuda.synchronize()
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=st):
            body()
        L, tab = list(p.lens), p.table.copy()
        for step in range(4):
            for s in range(3):
                L[s] += 1
                if tab[s, (L[s] - 1) // 64] < 0:
                    tab[s, (L[s] - 1) // 64] = free.pop()
            nk, nv, nq = (p.rng.standard_normal((3, h, hd)).astype(np.float32) for h in (KV, KV, H))
            for s in range(3):
                p.k[s] = np.concatenate([p.k[s], nk[s:s + 1]]); p.v[s] = np.concatenate([p.v[s], nv[s:s + 1]])
            with t.cuda.stream(st):
                lens.copy_(t.tensor(L, dtype=t.int32)); table.copy_(t.from_numpy(tab))
                q.copy_(t.from_numpy(nq.reshape(3, -1))); k.copy_(t.from_numpy(nk.reshape(3, -1))); v.copy_(t.from_numpy(nv.reshape(3, -1)))
                g.replay()
            st.synchronize()
            got = ctx.cpu().numpy()
            for s in range(3):
                want, tol = attend64(quant(p.k[s])[0], quant(p.v[s])[0], nq[s:s + 1], [L[s] - 1], H // KV)
                check(got[s:s + 1], want, tol)
            p.table, p.lens = tab, list(L)
            if step == 1:
                eager = p.attend(nq, H, [1, 1, 1], max_len=64 * p.ld)
                assert eager.tobytes() == got.tobytes()
        del g
    finally:
        gpu._ck(gpu.lib().moty_cuda_scratch_freeze(0, 0))
    p.status()


@pytest.mark.parametrize("rows", [1, 3, 70])
def test_attend_over_memory_that_holds_anything(gpu, t, rows):
    """The caller's memory is not zero: what lies behind the last position (infinite and NaN steps among it) has no effect."""
    H, KV, hd, L = 8, 2, 64, 150
    mem = t.full((5, gpu.Kv4.page_bytes(1, KV, hd)), 0xff, device="cuda", dtype=t.uint8)
    mem.view(t.int16)[1:] = 0x7c00
    p = Pool(gpu, t, KV, hd, [L], seed=13, pages=5)
    p.kv.close()
    p.kv = gpu.Kv4(1, KV, hd, 5, mem_ptr=mem.data_ptr())
    p.store()
    q = p.rng.standard_normal((rows, H, hd)).astype(np.float32)
    got = p.attend(q, H, [rows])
    want, tol = attend64(quant(p.k[0])[0], quant(p.v[0])[0], q, np.arange(L - rows, L), H // KV)
    check(got, want, tol)
