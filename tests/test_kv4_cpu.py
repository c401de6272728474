"""CPU: the paged 4-bit KV cache without a GPU -- the index arithmetic that the kernels share (compiled here with the host
compiler), the page bookkeeping, and the refusals of the C entries."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "moty_b200", "csrc")

HARNESS = r"""
#include "kv4_index.h"
#include <string.h>
extern "C" {
// marks every byte that the positions of one unit own; -1 when two pieces overlap or one leaves the unit
int unit_map(int hd) {
    std::vector<int> hits(kv4_unit_bytes(hd) * 2, 0);           // one entry per nibble
    for (int t = 0; t < KV4_PAGE; t++)
        for (int d = 0; d < hd; d++) {
            const int g = d / 32, kb = kv4_k_word(hd, t, g, (d >> 3) & 3), vb = kv4_v_piece(hd, t, g, (d >> 2) & 7);
            const int kn = 2 * kb + (d & 7), vn = 2 * vb + (d & 3);
            if (kn < 0 || kn >= 2 * kv4_k_step_off(hd) || vn < 2 * kv4_v_code_off(hd) || vn >= 2 * kv4_v_step_off(hd)) return -1;
            if (hits[kn]++ || hits[vn]++) return -1;
        }
    for (int i = 0; i < KV4_PAGE * (hd / 32); i++)
        for (int k = 0; k < 4; k++) {
            const int a = 2 * kv4_k_step_off(hd) + 4 * i + k, b = 2 * kv4_v_step_off(hd) + 4 * i + k;
            if (b >= (int)hits.size() || hits[a]++ || hits[b]++) return -1;
        }
    for (int h : hits) if (h != 1) return -1;
    return 0;
}
long long unit_off(int layers, int KV, int hd, int pages, int page, int layer, int head) {
    Kv4Geom g{layers, KV, hd, pages};
    if (!kv4_page_ok(g, page)) return -1;
    return (long long)kv4_unit_off(g, page, layer, head);
}
int row(int nseq, int rows, int ld, const int *row0, const int *len, int r, int *seq, int *pos) {
    Kv4Batch b{nseq, rows, ld, row0, len, nullptr};
    return kv4_row(b, r, seq, pos);
}
int seq(int nseq, int rows, int ld, const int *row0, const int *len, int s, int *r0, int *n, int *L) {
    Kv4Batch b{nseq, rows, ld, row0, len, nullptr};
    return kv4_seq(b, s, r0, n, L);
}
Kv4Pages *pages_new(int n) { auto *p = new Kv4Pages(); p->init(n); return p; }
void pages_del(Kv4Pages *p) { delete p; }
int pages_alloc(Kv4Pages *p, int n, int *out) { return p->alloc(n, out); }
int pages_retain(Kv4Pages *p, int n, const int *ids) { return p->retain(ids, n); }
int pages_release(Kv4Pages *p, int n, const int *ids) { return p->release(ids, n); }
int pages_free(Kv4Pages *p) { return p->free_count(); }
int pages_refs(Kv4Pages *p, int id) { return p->refs[id]; }
int pages_compact(Kv4Pages *p, int *src, int *dst) {
    std::vector<int> s, d; p->plan(&s, &d);
    for (size_t i = 0; i < s.size(); i++) { src[i] = s[i]; dst[i] = d[i]; }
    p->moved(s, d);
    return (int)s.size();
}
}
"""


@pytest.fixture(scope="module")
def h(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4")
    src, so = str(d / "h.cpp"), str(d / "h.so")
    with open(src, "w") as f:
        f.write(HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, src, "-o", so], check=True)
    L = C.CDLL(so)
    L.unit_off.restype = C.c_longlong
    L.pages_new.restype = C.c_void_p
    return L


def _i(a):
    a = np.ascontiguousarray(a, np.int32)
    return a, a.ctypes.data_as(C.POINTER(C.c_int))


@pytest.mark.parametrize("hd", range(32, 257, 32))
def test_unit_layout_covers_every_nibble_once(h, hd):
    assert h.unit_map(hd) == 0


def test_unit_offsets(h):
    """Every unit of the largest pools starts inside them, offsets past 32 bits included; pages outside are refused."""
    for layers, KV, hd, pages in ((1, 1, 32, 1), (64, 16, 256, 3000), (28, 8, 128, 1 << 25)):
        page = layers * KV * 72 * hd
        for p in (0, pages // 2, pages - 1):
            for l, k in ((0, 0), (layers - 1, KV - 1)):
                off = h.unit_off(layers, KV, hd, pages, p, l, k)
                assert off == p * page + (l * KV + k) * 72 * hd and off + 72 * hd <= pages * page
        for p in (-1, -2, pages, 2**31 - 1, -2**31):
            assert h.unit_off(layers, KV, hd, pages, p, 0, 0) == -1


def test_rows_of_a_batch(h):
    row0, pr = _i([0, 1, 1, 4, 9]); ln, pl = _i([5, 7, 3, 700])
    want = [(0, 4), (2, 0), (2, 1), (2, 2), (3, 695), (3, 696), (3, 697), (3, 698), (3, 699)]
    s, p = C.c_int(), C.c_int()
    for r in range(12):
        st = h.row(4, 12, 11, pr, pl, r, C.byref(s), C.byref(p))
        if r < 9:
            assert st == 1 and (s.value, p.value) == want[r]
        else:
            assert st == 0                       # behind the last sequence


def test_rows_of_arrays_that_are_no_batch(h):
    """Whatever the arrays hold, a row that is accepted has a position inside its table and its sequence inside the batch."""
    rng = random.Random(0)
    s, p, r0, n, L = (C.c_int() for _ in range(5))
    wild = [-2**31, -5, -1, 0, 1, 2, 3, 63, 64, 65, 100, 2**31 - 1]
    for _ in range(4000):
        nseq, rows, ld = rng.randint(1, 5), rng.randint(1, 9), rng.randint(1, 3)
        row0, pr = _i([rng.choice(wild) for _ in range(nseq + 1)]); ln, pl = _i([rng.choice(wild) for _ in range(nseq)])
        for r in range(rows):
            if h.row(nseq, rows, ld, pr, pl, r, C.byref(s), C.byref(p)) == 1:
                assert 0 <= s.value < nseq and 0 <= p.value < ld * 64 and row0[s.value] <= r < row0[s.value + 1]
        for q in range(nseq):
            if h.seq(nseq, rows, ld, pr, pl, q, C.byref(r0), C.byref(n), C.byref(L)) == 1:
                assert 0 <= r0.value and n.value > 0 and r0.value + n.value <= rows and n.value <= L.value <= ld * 64


@pytest.mark.parametrize("nseq", [1, 2, 15, 16, 17, 64, 255, 256, 257, 5000])
def test_rows_of_many_sequences(h, nseq):
    """Every row finds its sequence among many, empty ones among them; offsets that do not ascend stay inside the arrays."""
    rng = random.Random(nseq)
    n = [rng.choice([0, 0, 1, 1, 2, 5]) for _ in range(nseq)]
    off = [0]
    for x in n:
        off.append(off[-1] + x)
    rows, ld = off[-1] + 3, 4
    row0, pr = _i(off); ln, pl = _i([x + rng.randint(0, 200) for x in n])
    s, p = C.c_int(), C.c_int()
    at = 0
    for r in range(rows):
        while at < nseq and r >= off[at + 1]:
            at += 1
        st = h.row(nseq, rows, ld, pr, pl, r, C.byref(s), C.byref(p))
        if at == nseq:
            assert st == 0
        else:
            assert st == 1 and s.value == at and p.value == ln[at] - n[at] + r - off[at]
    wild, pw = _i([rng.choice([-7, 0, 1, rows, 1 << 30, rng.randint(0, rows)]) for _ in range(nseq + 1)])
    for r in range(rows):
        st = h.row(nseq, rows, ld, pw, pl, r, C.byref(s), C.byref(p))
        assert 0 <= s.value < nseq
        if st == 1:
            assert wild[s.value] <= r < wild[s.value + 1] and 0 <= p.value < ld * 64


def test_page_books(h):
    rng = random.Random(1)
    N = 40
    p = C.c_void_p(h.pages_new(N))
    held = []                                    # every owner's id
    for step in range(600):
        kind = rng.random()
        if kind < 0.4:
            n = rng.randint(0, 7)
            a, pa = _i(np.zeros(n + 1)); free = h.pages_free(p)
            ok = h.pages_alloc(p, n, pa)
            assert ok == (n <= free)
            if ok:
                ids = [int(v) for v in a[:n]]
                lowest = sorted(set(range(N)) - set(held))[:n]
                assert ids == lowest
                held += ids
        elif kind < 0.55 and held:
            ids = [rng.choice(held) for _ in range(rng.randint(1, 4))] + [-1]
            assert h.pages_retain(p, len(ids), _i(ids)[1]); held += ids[:-1]
        elif kind < 0.93 and held:
            rng.shuffle(held); n = rng.randint(1, min(6, len(held)))
            assert h.pages_release(p, n + 1, _i([-1] + held[:n])[1]); held = held[n:]
        else:
            a, pa = _i(np.zeros(N)); b, pb = _i(np.zeros(N))
            n = h.pages_compact(p, pa, pb)
            src, dst = [int(v) for v in a[:n]], [int(v) for v in b[:n]]
            live = set(held)
            assert src == sorted(src) and dst == sorted(dst) and not set(src) & set(dst)
            ren = dict(zip(src, dst)); held = [ren.get(v, v) for v in held]
            assert set(held) == set(range(len(live)))
        assert h.pages_free(p) == N - len(set(held))
        for i in range(N):
            assert h.pages_refs(p, i) == held.count(i)
        # refusals leave the books alone
        free_id = next((i for i in range(N) if i not in held), None)
        for bad in ([N], [-2], [free_id] if free_id is not None else [N]):
            assert not h.pages_retain(p, 1, _i(bad)[1]) and not h.pages_release(p, 1, _i(bad)[1])
        if held:
            v = held[0]
            assert not h.pages_release(p, held.count(v) + 1, _i([v] * (held.count(v) + 1))[1])
    h.pages_del(p)


def test_refusals_without_a_gpu():
    import moty_b200 as mb
    for layers, KV, hd in ((0, 1, 64), (1, 0, 64), (1, 1, 0), (1, 1, 48), (1, 1, 288), (1, 1, -32), (70000, 1, 64)):
        with pytest.raises(mb.MotyCudaError, match="head_dim"):
            mb.Kv4.page_bytes(layers, KV, hd)
        with pytest.raises(mb.MotyCudaError, match="head_dim"):
            mb.Kv4(layers, KV, hd, 4)
    assert mb.Kv4.page_bytes(28, 8, 128) == 28 * 8 * 72 * 128
    with pytest.raises(mb.MotyCudaError, match="pages="):
        mb.Kv4(1, 1, 64, 0)
    with pytest.raises(mb.MotyCudaError, match="128-byte"):
        mb.Kv4(1, 1, 64, 4, mem_ptr=64)
    L = mb.lib()
    b = mb.Kv4Batch(1, 1, 16, 16, 16, 1)
    assert L.moty_cuda_kv4_append_dev(None, 0, 16, 16, 0, b.ptr, None) == -2
    assert L.moty_cuda_kv4_fetch_dev(None, 0, 16, 16, b.ptr, None) == -2
    assert L.moty_cuda_kv4_attend_dev(None, 0, 16, 16, 0, 1, 0, 0.0, b.ptr, None) == -2
    assert L.moty_cuda_kv4_fork_dev(None, 1, 16, 16, 16, 1, 16, 16, 1, None) == -2
    assert L.moty_cuda_kv4_compact_dev(None, 1, 16, 16, 0, None, None, None) == -2
    n = C.c_int()
    assert L.moty_cuda_kv4_alloc(None, 1, C.byref(n)) == -2 and L.moty_cuda_kv4_compact_plan(None, 0, None, None, C.byref(n)) == -2
    assert L.moty_cuda_kv4_free(None) == 0
