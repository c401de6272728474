"""GPU: the paged 4-bit KV cache where attention's sums are hard -- one position that takes nearly all the weight and holds
nothing, groups of dims far smaller than the others, long sums of one sign -- and the corners of calls, forks and moves.

Scores here are exact: a query row holds a single 1, a key row a single value of few bits, so that a score is that value.
What is left, with e = 2^-24 and scores that span `gap` (natural units):
  * a weight: scale and log2(e) as f32 2 e gap, the exponent's rounding e (gap + 11) (base-2 arguments end 16 below or above
    their reference), exp2 4 e; numerator and denominator, and joins by two more exp2:  (6 gap + 46) e;
  * weight, step and value as 16-bit pieces, the quotient: 8 e;
  * sums of at most 64 products in a matrix unit, which cuts them off, 2 e each: 128 e; then f32 sums of at most T / 16
    roundings, each at random e of what is there so far (the values' signs are random: three times the root of half of them).
|error| <= e (6 gap + 182 + 3 sqrt(T / 32)) |result|, in the 2-norm over the 32 dims of a group: of every group by itself.
"""
import ctypes as C
import math

import numpy as np
import pytest

from test_gpu_kv4 import Pool, attend64, check, quant

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(scope="module")
def t():
    import torch
    torch.backends.cuda.matmul.allow_tf32 = False
    return torch


# (query heads, rows a sequence, head width): decode of four and of eight columns, the prompt kernels of matrix instructions
# (32, 160, 256) and of tensor memory (64 to 128).  40 sequences of 8 KV heads share one table: a CTA walks many pages.
KERNELS = [(8, 1, 32), (8, 1, 128), (8, 1, 256), (64, 1, 64), (64, 1, 128), (16, 4, 224), (32, 20, 32), (32, 20, 160), (32, 20, 256),
           (32, 20, 64), (32, 20, 96), (32, 20, 128)]
NSEQ, KV = 40, 8


def hard(gpu, t, H, rows, hd, T, scores, values, window=0):
    """Attention of NSEQ sequences over one, and what it should be for some of the rows: (got, want) [n][hd], the scores' span."""
    p = Pool(gpu, t, KV, hd, [T], seed=H * hd + rows + T)
    rng = p.rng
    s = rng.integers(0, 3, T) / 8                            # "even"
    if scores.startswith("sink"):                            # position 0 stands far above the others, and holds nothing
        s[0] = float(scores[4:])
    elif scores == "ragged":                                 # pages of very different weight
        s = np.round(rng.standard_normal(T) * 48) / 8 + 4 * np.round(rng.standard_normal(T // 64 + 1))[np.arange(T) // 64]
    p.k[0][:] = 0; p.k[0][:, :, 0] = s[:, None]
    if scores.startswith("sink"):
        p.v[0][0] = 0
    if values == "small":
        p.v[0] *= np.float32(2**-6)
    if values == "groups":                                   # the last group's values are 2^14 times smaller
        p.v[0] *= np.float32(2**-4); p.v[0][:, :, hd - 32:] *= np.float32(2**-14)
    p.store()
    q = np.zeros((NSEQ * rows, H, hd), np.float32); q[:, :, 0] = 1
    got = p.attend(q, H, [rows] * NSEQ, window=window, scale=1.0, lens=[T] * NSEQ, table=np.repeat(p.table, NSEQ, 0)).reshape(NSEQ, rows, H, hd)
    p.status()
    k, v = quant(p.k[0])[0], quant(p.v[0])[0]
    assert np.array_equal(k[:, 0, 0], s) and not k[:, :, 1:].any()
    a, b = [], []
    for i, r, h in [(0, 0, 0), (0, rows - 1, H - 1), (NSEQ - 1, rows // 2, H // 2), (NSEQ // 2, rows - 1, 1)]:
        pos = T - rows + r
        lo = max(0, pos - window + 1) if window else 0
        w = np.exp(s[lo:pos + 1] - s[lo:pos + 1].max())
        a.append(got[i, r, h]); b.append(w @ v[lo:pos + 1, h // (H // KV)] / w.sum())
    return np.array(a), np.array(b), float(s.max() - s.min())


def group_errors(got, want):
    d = (got - want).reshape(len(want), -1, 32)
    return np.linalg.norm(d, axis=-1) / np.linalg.norm(want.reshape(d.shape), axis=-1)


@pytest.mark.parametrize("T", [70, 2065, 5000])
@pytest.mark.parametrize("scores,values", [("sink10", "plain"), ("sink14", "plain"), ("sink14", "small"), ("even", "groups"), ("ragged", "small")])
@pytest.mark.parametrize("H,rows,hd", KERNELS)
def test_attend_small_weights_and_small_values_keep_their_bits(gpu, t, H, rows, hd, scores, values, T):
    if values == "groups" and hd == 32:
        values = "small"                                     # (one group)
    got, want, gap = hard(gpu, t, H, rows, hd, T, scores, values)
    assert group_errors(got, want).max() <= E * (6 * gap + 182 + 3 * math.sqrt(T / 32))


@pytest.mark.parametrize("H,KV,nseq,rows,hd", [(8, 2, 80, 20, 32), (8, 2, 80, 20, 256)])
def test_attend_prompts_with_long_sums_of_one_sign(gpu, t, H, KV, nseq, rows, hd):
    """Weights of three sizes and positive values: every sum grows evenly, and additions to a large sum round the same way
    again and again.  Sums of at most 64 passes and of 1024 positions each (T / 1024 of them) err by e a step at most, a
    pass's products by 8 e, numerator and denominator; weights and pieces by (6 gap + 54) e."""
    T = 66000
    p = Pool(gpu, t, KV, hd, [T], seed=hd)
    s = p.rng.integers(0, 3, T) / 8
    p.k[0][:] = 0; p.k[0][:, :, 0] = s[:, None]
    p.v[0] = np.abs(p.v[0]) + np.float32(0.5)
    p.store()
    q = np.zeros((nseq * rows, H, hd), np.float32); q[:, :, 0] = 1
    got = p.attend(q, H, [rows] * nseq, scale=1.0, lens=[T] * nseq, table=np.repeat(p.table, nseq, 0)).reshape(nseq, rows, H, hd)
    p.status()
    v = quant(p.v[0])[0]
    for i, r, h in [(0, 0, 0), (nseq - 1, rows - 1, H - 1)]:
        w = np.exp(s[:T - rows + r + 1] - 0.25)
        want = w @ v[:T - rows + r + 1, h // (H // KV)] / w.sum()
        assert np.abs(got[i, r, h] / want - 1).max() <= E * (2 * (8 + 64 + T / 1024) + 6 * 0.25 + 54)


@pytest.mark.parametrize("H,rows,hd", [(8, 1, 32), (8, 1, 96), (64, 1, 128), (16, 1, 256), (32, 20, 32), (32, 20, 64), (32, 20, 128), (32, 20, 256)])
def test_attend_of_one_position_is_its_values(gpu, t, H, rows, hd):
    """A row that sees a single position, of a score without rounding, is that position's value row, to the bit: the first
    positions of sequences, and rows with a window of one.  (Activations are quantised after this: values of few bits lie on ties there.)  Scores are exact in
    the kernels' base-2 units: eighths, scaled by what is 1 after log2(e)."""
    T, log2e = 150, np.float32(1.44269504)
    scale = np.float32(1) / log2e
    assert np.float32(scale * log2e) == 1
    p = Pool(gpu, t, KV, hd, [T], seed=hd + rows)
    p.k[0][:] = 0; p.k[0][:, :, 0] = p.rng.integers(-40, 41, (T, 1)) / 8
    p.store()
    q = np.zeros((NSEQ * rows, H, hd), np.float32); q[:, :, 0] = 1
    v = quant(p.v[0])[0].astype(np.float32)
    G = H // KV
    got = p.attend(q, H, [rows] * NSEQ, scale=float(scale), window=1, lens=[T] * NSEQ, table=np.repeat(p.table, NSEQ, 0), max_len=T).reshape(NSEQ, rows, H, hd)
    want = np.repeat(v[T - rows:], G, 1)
    assert np.array_equal(got, np.broadcast_to(want, got.shape))
    # the first `rows` positions of a sequence: its row 0 sees position 0 alone
    got = p.attend(q, H, [rows] * NSEQ, scale=float(scale), lens=[rows] * NSEQ, table=np.repeat(p.table, NSEQ, 0), max_len=p.ld * 64).reshape(NSEQ, rows, H, hd)
    assert np.array_equal(got[:, 0], np.broadcast_to(np.repeat(v[0], G, 0), got[:, 0].shape))
    p.status()


@pytest.mark.parametrize("hd", [64, 128])
def test_attend_prompts_weights_total_over_a_long_span(gpu, t, hd):
    """The tensor-memory kernel's span of 512 pages, weights that hardly differ, values that are all the same: the result is the
    value.  The weights' total is summed over 32 positions, 16 pages and 32 such parts; additions to a sum err by e at most, all
    the same way where the sum grows evenly, by half of that on the average and of half the final sum:  (32 + 16 + 32) e / 4.
    The 512 pages' outputs round at random, 0.58 e sqrt(512 / 3), and 12 products' sums are cut off by e / 2 on the average."""
    T, rows, nseq, H, KV = 32700, 20, 80, 8, 2
    p = Pool(gpu, t, KV, hd, [T], seed=hd)
    p.k[0][:] = 0; p.k[0][:, :, 0] = p.rng.integers(0, 3, (T, 1)) / 1024
    p.v[0][:] = 1.3
    p.store()
    q = np.zeros((nseq * rows, H, hd), np.float32); q[:, :, 0] = 1
    got = p.attend(q, H, [rows] * nseq, scale=1.0, lens=[T] * nseq, table=np.repeat(p.table, nseq, 0)).astype(np.float64)
    p.status()
    assert abs(np.mean(got / quant(p.v[0])[0][0, 0, 0]) - 1) <= E * (20 + 0.58 * math.sqrt(512 / 3) + 6)


# windows that leave rows with one page, with a page's end inside, with all; absent pages in front of, inside and behind them.  Key
# values of sequences' own tables differ by where pages are missing only.
@pytest.mark.parametrize("H,hd", [(32, 64), (32, 96), (32, 128), (32, 32), (32, 256)])
@pytest.mark.parametrize("window", [0, 1, 30, 64, 100, 700])
def test_attend_prompts_windows_absent_pages_and_rows_that_are_not_finite(gpu, t, H, hd, window):
    """Prompt kernels (tensor memory at 64 to 128): every mask at once, against the 64-bit form; a query row with an infinity or a
    NaN is NaN where it sees anything and 0 where it sees nothing, and changes no other row."""
    T, rows, G = 420, 40, H // KV
    p = Pool(gpu, t, KV, hd, [T], seed=hd + window, scale=2.0, extra_ld=3)
    table = np.repeat(p.table, NSEQ, 0)
    absent = {s: [] for s in range(NSEQ)}
    absent[1] = [6]; absent[2] = [5, 6]; absent[3] = [0, 3, 4]; absent[4] = list(range(7)); absent[5] = [1, 2, 5]
    for s, gone in absent.items():
        table[s, gone] = -1
    q = p.rng.standard_normal((NSEQ, rows, H, hd)).astype(np.float32)
    for s in range(6):
        q[s, 3, 5, 1] = np.nan; q[s, 17, 0, hd - 1] = np.inf; q[s, rows - 1, H - 1, 0] = -np.inf; q[s, 25, 9] = np.nan
    got = p.attend(q, H, [rows] * NSEQ, window=window, lens=[T] * NSEQ, table=table).reshape(NSEQ, rows, H, hd)
    p.status()
    k, v = quant(p.k[0])[0], quant(p.v[0])[0]
    for s in (0, 1, 2, 3, 4, 5, NSEQ - 1):
        hidden = np.isin(np.arange(T) // 64, absent[s])
        for r in (0, 3, 4, 17, 25, 35, 36, rows - 1):
            pos = T - rows + r
            for h in {0, 5, 9, H - 1}:
                g = h // G
                lo = max(0, pos - window + 1) if window else 0
                fin = np.isfinite(q[s, r, h]).all()
                if hidden[lo:pos + 1].all():
                    assert (got[s, r, h] == 0).all()
                elif not fin:
                    assert np.isnan(got[s, r, h]).all()
                else:
                    want, tol = attend64(k[:, g:g + 1], v[:, g:g + 1], q[s, r:r + 1, h:h + 1], [pos], 1, window, hidden=hidden)
                    check(got[s, r:r + 1, h:h + 1], want, tol)


@pytest.mark.parametrize("rows,lens", [(1, [300, 200]), (40, [300, 200]), (40, [2000, 1900]), (2, [9000, 5000])])
@pytest.mark.parametrize("what", ["len_past_table", "rows_more_than_len"])
def test_rows_behind_a_refused_sequence_stay(gpu, t, rows, lens, what):
    """The last sequence is refused: its rows become 0 (attend) or stay (fetch), the rows behind it stay, the first sequence's
    come out as always -- in one launch and with spans joined in a second."""
    H, hd, pad = 4, 64, 5
    p = Pool(gpu, t, 2, hd, lens, seed=rows)
    q = p.rng.standard_normal((2 * rows + pad, H, hd)).astype(np.float32)
    good = p.attend(q[:2 * rows], H, [rows, rows])
    bad = [lens[0], 64 * p.ld + 1 if what == "len_past_table" else rows - 1]
    got = p.attend(q, H, [rows, rows], pad=pad, lens=bad, max_len=max(lens))
    with pytest.raises(gpu.MotyCudaError, match="4-bit KV"):
        p.status()
    assert got[:rows].tobytes() == good[:rows].tobytes() and (got[rows:2 * rows] == 0).all() and (got[2 * rows:] == 7).all()
    b = p.batch([rows, rows], lens=bad, pad=pad, max_len=max(lens))
    k = t.full((2 * rows + pad, 2 * hd), 5.0, device="cuda"); v = k.clone()
    p.kv.fetch_dev(0, k.data_ptr(), v.data_ptr(), b, stream=p.sh())
    t.cuda.synchronize()
    with pytest.raises(gpu.MotyCudaError, match="4-bit KV"):
        p.status()
    for x, held in ((k, p.k[0]), (v, p.v[0])):
        assert (x[rows:] == 5).all()
        assert np.array_equal(x[:rows].cpu().numpy().reshape(rows, 2, hd), quant(held[lens[0] - rows:])[0].astype(np.float32))


@pytest.mark.parametrize("src,dst,made", [([5, 4], [0, 1], {5: 0}), ([4, 5], [1, 0], {4: 1}), ([4, 5], [1, 1], {4: 1}), ([3, 5], [0, 3], {3: 0}), ([-1, 5], [0, 1], {5: 1}),
                                          ([4, 5], [-2, 1], {5: 1}), ([4, 5], [8, 9], {}), ([4, 5], [0, 1], {4: 0, 5: 1})])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_move_that_is_refused_renames_nothing(gpu, t, src, dst, made, in_place):
    """Entries follow the pages that were copied, and no others: lists out of order, that meet, or that leave the pool."""
    layers, heads, hd, pages = 2, 1, 64, 8
    g = t.Generator(device="cuda").manual_seed(5)
    mem = t.randint(0, 256, (pages, gpu.Kv4.page_bytes(layers, heads, hd)), generator=g, device="cuda", dtype=t.uint8)
    before = mem.cpu().numpy()
    kv = gpu.Kv4(layers, heads, hd, pages, mem_ptr=mem.data_ptr())
    d = lambda a: t.tensor(a, device="cuda", dtype=t.int32)
    S, D, T = d(src), d(dst), d([-1, 4, 5, 3, 0, 7, 5, 4, -1])
    want = [made.get(int(x), int(x)) for x in T.cpu()]
    out = T if in_place else t.full_like(T, 99)
    sh = gpu.stream_handle(t.cuda.current_stream())
    kv.compact_dev(2, S.data_ptr(), D.data_ptr(), T.numel(), T.data_ptr(), out.data_ptr(), stream=sh)
    t.cuda.synchronize()
    assert gpu.lib().moty_cuda_kernel_status(0, sh) == (0 if len(made) == 2 else -6)
    assert out.cpu().tolist() == want
    after = mem.cpu().numpy()
    for a, b in made.items():
        assert np.array_equal(after[b], before[a])


@pytest.mark.parametrize("lens,new,sound", [
    ([70, 100], [5, 1], [0]),                    # into the page that the first fork copies from
    ([70, 100], [3, 6], [1]),                    # into the page that the second copies from
    ([70, 100], [1, 6], [1]), ([70, 100], [5, 3], [0]),      # into its own source's last page
    ([70, 100], [3, 1], []),                     # each into the other's
    ([70, 128], [5, 1], [0, 1]),                 # a source that ends with its page takes no fresh one: whatever is given is not used
    ([70, 100], [0, 2], [0, 1]),                 # (pages in front of the last ones are not read: which pages are free is the caller's to know)
])
def test_forks_into_a_page_that_is_copied_are_refused(gpu, t, lens, new, sound):
    layers, heads, hd, pages, ld = 2, 1, 64, 8, 3
    g = t.Generator(device="cuda").manual_seed(2)
    mem = t.randint(0, 256, (pages, gpu.Kv4.page_bytes(layers, heads, hd)), generator=g, device="cuda", dtype=t.uint8)
    before = mem.cpu().numpy()
    kv = gpu.Kv4(layers, heads, hd, pages, mem_ptr=mem.data_ptr())
    table = np.full((4, ld), -1, np.int32); table[0, :2] = [0, 1]; table[1, :2] = [2, 3]
    ln = np.array(lens + [0, 0], np.int32)
    d = lambda a: t.tensor(a, device="cuda", dtype=t.int32)
    S, D, N, T, L = d([0, 1]), d([2, 3]), d(new), d(table), d(ln)
    sh = gpu.stream_handle(t.cuda.current_stream())
    kv.fork_dev(2, S.data_ptr(), D.data_ptr(), N.data_ptr(), 4, L.data_ptr(), T.data_ptr(), ld, stream=sh)
    t.cuda.synchronize()
    assert gpu.lib().moty_cuda_kernel_status(0, sh) == (0 if len(sound) == 2 else -6)
    want, wl = before.copy(), ln.copy()
    for f in sound:
        tail = lens[f] % 64 > 0
        table[2 + f] = table[f]; wl[2 + f] = lens[f]
        if tail:
            want[new[f]] = before[table[f, lens[f] // 64]]; table[2 + f, lens[f] // 64] = new[f]
    assert np.array_equal(mem.cpu().numpy(), want) and np.array_equal(T.cpu().numpy(), table) and np.array_equal(L.cpu().numpy(), wl)


def test_calls_from_a_thread_with_a_context_of_the_driver_api(gpu, t):
    """A thread whose current context on the device is not the primary one: the library's calls run in theirs all the same."""
    import threading

    p = Pool(gpu, t, 2, 64, [100], seed=3)
    q = p.rng.standard_normal((1, 4, 64)).astype(np.float32)
    want = p.attend(q, 4, [1])
    b, qd, ctx = p.batch([1]), p.dev(q, np.float32), t.zeros((1, 256), device="cuda")
    t.cuda.synchronize()
    cu = C.CDLL("libcuda.so.1")
    failed = []

    def work():
        try:
            dev, own = C.c_int(), C.c_void_p()
            assert cu.cuDeviceGet(C.byref(dev), 0) == 0 and cu.cuCtxCreate_v2(C.byref(own), 0, dev) == 0
            try:
                p.kv.attend_dev(0, ctx.data_ptr(), qd.data_ptr(), 4, b)            # (the library's own stream)
                gpu.sync(0)
                more = gpu.Kv4(1, 1, 32, 2)
                more.close()
            finally:
                assert cu.cuCtxDestroy_v2(own) == 0
        except BaseException as e:
            failed.append(e)

    th = threading.Thread(target=work)
    th.start(); th.join()
    assert not failed, failed
    assert ctx.cpu().numpy().tobytes() == want.tobytes()
    assert np.array_equal(p.attend(q, 4, [1]), want)
    p.status()
