"""CPU: what the paged 4-bit KV cache's kernels rely on that no result shows, and its decoder's books when a step fails."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "moty_b200", "csrc")


def test_roles_take_their_registers_in_their_own_branch():
    """A warpgroup's register count is set as the first statement of a branch that whole warpgroups take: only there is the
    code that follows bounded by it.  The shares add up to what the block is launched with."""
    src = open(os.path.join(CSRC, "kv4_prompt_tc.cu")).read()
    assert len(re.findall(r"setmaxnreg\.(?:inc|dec)", src)) == 2                   # in role_registers alone
    calls = re.findall(r"(if \(warp >= \d+\)|else) \{\n\s*role_registers<(true|false), (\w+)>\(\);", src)
    assert len(calls) == len(re.findall(r"role_registers<(?:true|false)", src)) == 3
    value = lambda name: int(re.search(rf"{name} = (\d+)", src).group(1))
    edge, total = value("PT_T") // 32, 0
    for cond, more, regs in calls:
        low = int(re.search(r"\d+", cond).group()) if cond != "else" else 0
        assert low % 4 == 0 and (more == "true") == (value(regs) > value("PT_REGS"))
        total += (edge - low) * 32 * value(regs); edge = low
    assert edge == 0 and total <= value("PT_T") * value("PT_REGS") <= 65536


def test_rows_behind_a_refused_sequence_are_nobodys(tmp_path):
    """Rows behind the last sequence belong to none, also where that sequence is refused (a length past its table): only its own
    rows count as refused."""
    src, so = str(tmp_path / "r.cpp"), str(tmp_path / "r.so")
    with open(src, "w") as f:
        f.write('#include "kv4_index.h"\nextern "C" int row(int nseq, int rows, int ld, const int *row0, const int *len, int r) {\n'
                "    Kv4Batch b{nseq, rows, ld, row0, len, nullptr}; int s, p; return kv4_row(b, r, &s, &p); }\n")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, src, "-o", so], check=True)
    lib = C.CDLL(so)
    arr = lambda a: (C.c_int * len(a))(*a)
    none, ok, bad, stray = 0, 1, 2, 3
    look = lambda row0, lens, rows, ld=2: [lib.row(len(lens), rows, ld, arr(row0), arr(lens), r) for r in range(rows)]
    assert look([0, 2, 5], [9, 9], 8) == [ok] * 5 + [none] * 3
    assert look([0, 2, 5], [9, 129], 8) == [ok] * 2 + [bad] * 3 + [stray] * 3
    assert look([0, 2, 5], [129, 9], 8) == [bad] * 2 + [ok] * 3 + [none] * 3
    assert look([1, 3, 2], [9, 9], 5) == [none, ok, ok, stray, stray]              # the second ends before it begins
    assert look([0, 9], [20], 5) == [bad] * 5                                      # ends behind the buffers


def test_prompts_fall_back_where_the_tensor_memory_kernel_cannot_run(tmp_path):
    """How a call is cut when that kernel was built with other registers than its roles share out: the other prompt kernel's
    tiles, for every call that would have gone to it."""
    import moty_b200 as mb
    src, exe = str(tmp_path / "p.cpp"), str(tmp_path / "p")
    with open(src, "w") as f:
        f.write(r'''
#include "kv4_attend.cuh"
#include <cstdio>
int main() {
    int seen = 0;
    for (int hd : {32, 64, 96, 128, 160, 256})
        for (int rows : {1, 20, 400, 4096})
            for (int len : {4096, 40000}) {
                Kv4Attend a{};
                a.geo = Kv4Geom{1, 8, hd, 100}; a.b.nseq = 2; a.b.rows = 2 * rows; a.b.ld = 1000;
                a.H = 32; a.G = 4; a.max_rows = rows; a.max_len = len;
                a.tc = true;
                const Kv4Plan p = kv4_plan(a, 148);
                a.tc = false;
                const Kv4Plan q = kv4_plan(a, 148);
                seen += p.tc;
                if (q.tc || q.decode != p.decode || q.span % KV4_PAGE || (long long)q.span * q.nsplit < len) return 1;
                if (p.tc ? q.cols != KV4_LINES || (long long)q.ntile * KV4_LINES < 4LL * rows
                         : q.cols != p.cols || q.ntile != p.ntile || q.span != p.span || q.nsplit != p.nsplit) return 2;
            }
    printf("%d\n", seen);
    return 0;
}
''')
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", CSRC, "-I", os.path.join(ROOT, "include"), "-I", "/usr/local/cuda/include", src, mb.LIB_PATH,
                    "-L/usr/local/cuda/lib64", "-lcudart", "-Wl,-rpath," + os.path.dirname(mb.LIB_PATH), "-o", exe], check=True)
    assert int(subprocess.run([exe], check=True, capture_output=True, text=True).stdout) >= 6


@pytest.mark.parametrize("name", ["DenseDecoder", "GemmaDecoder", "PagedDecoder"])
def test_an_allocation_that_fails_leaves_no_room_behind(name):
    """Buffers for more rows that could not all be made: the decoder must not take the smaller ones that are left for them."""
    import types

    import torch
    from moty_b200 import decoder
    d = object.__new__(getattr(decoder, name))
    d.H, d.KV, d.hd, d.D, d._qw, d._kw = 4, 2, 32, 128, 128, 64
    d.head = types.SimpleNamespace(O=300)
    d.dev, left = "cpu", [99]

    def empty(*a, **k):
        left[0] -= 1
        if left[0] < 0:
            raise MemoryError
        return torch.empty(*a, **k)

    d.torch = types.SimpleNamespace(empty=empty, float32=torch.float32, int32=torch.int32)
    d._alloc(4)
    made = 99 - left[0]
    assert d.cap == 4
    for n in range(made):
        left[0] = n
        with pytest.raises(MemoryError):
            d._alloc(50)
        assert d.cap <= min(len(d.x), len(d.ctx), len(d.ids), len(d.nrm), len(d.tmp))
        left[0] = 99
        d._alloc(4)
        assert d.cap == 4
