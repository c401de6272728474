"""The paged 4-bit KV cache: its operators as a serving program calls them, in plain form and through the library.

The cache holds key and value rows of many sequences in pages of 64 positions.  A row of one KV head is cut into groups
of 32 dimensions that share one signed f16 step d; a value is code * d with a code of -8 .. 7:

    big   = the group's first value of largest magnitude,  other = the largest magnitude of the opposite sign
    step  = max(|big| / 8, other / 7)  in f32,   d = f16(big > 0 ? -step : step)
    code  = clamp(rint(x / d), -8, 7)            (0 where d is 0; the quotient rounded once, ties to even)

A batch is ragged: rows row0[s] .. row0[s + 1] - 1 belong to sequence s and are the LAST of its len[s] positions; its
pages are table[s][0 ..], -1 for a page that was freed.  The operators:

    append + fetch   quantise new key / value rows into the pages, and read the same rows back as the values held
    attend           softmax(q k / sqrt(hd)) v over a sequence's positions, causal, optionally the last `window` only
    fork             sequences that share a prefix: table rows copied, the last partial page copied
    compact          live pages moved to the low ids, the page table renamed
"""
import math
import random

import torch

own = False

PAGE, GROUP = 64, 32
DEV = "cuda"


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    def attend(name, nseq, rows, max_len, H, KV, hd, window=0, ragged=False, mix=1):
        return dict(name=name, op="attend", nseq=nseq, rows=rows, max_len=max_len, H=H, KV=KV, hd=hd, window=window,
                    ragged=ragged, mix=mix)

    return [
        # one user, one token, the head layout of the small dense model that the decode benchmark runs: latency
        attend("attend_one_1000", 1, 1, 1000, 16, 8, 128),
        # a serving step: 64 sequences of mixed length, 32 query heads on 8 KV heads
        attend("attend_batch_8k", 64, 1, 8192, 32, 8, 128, ragged=True, mix=2),
        # the sliding layers of the 256-wide-head model: a window of 1024, the pages before it freed
        attend("attend_window_hd256", 13, 1, 4500, 16, 8, 256, window=1024, ragged=True, mix=3),
        # one very long conversation of the routed model's layout: 32 query heads on 4 KV heads
        attend("attend_long_131k", 1, 1, 131072, 32, 4, 128),
        # chunked prefill beside running sequences: blocks of prompt and single tokens in one call, odd head width
        attend("attend_mixed_hd96", 9, 333, 2900, 20, 4, 96, ragged=True, mix=4),
        # a whole prompt
        attend("attend_prompt_4096", 1, 4096, 4096, 16, 8, 128),
        # the new rows of one decode step of 64 sequences
        dict(name="append_step_64", op="append", nseq=64, rows=1, max_len=4001, KV=8, hd=128, ragged=True, mix=5),
        # a prompt's rows for one layer, many heads (every query head with its own KV head)
        dict(name="append_prompt_4096", op="append", nseq=3, rows=4096, max_len=5000, KV=16, hd=128, ragged=True, mix=6),
        # one sequence forked into four samples, 28 layers
        dict(name="fork_4", op="fork", n=4, nsrc=1, max_len=777, layers=28, KV=8, hd=128, mix=7),
        # a beam step over many sequences
        dict(name="fork_48", op="fork", n=48, nsrc=16, max_len=640, layers=28, KV=8, hd=128, mix=8),
        # a few pages to move in a small pool, odd head width
        dict(name="compact_5", op="compact", n=5, pages=40, nseq=6, ld=16, layers=5, KV=3, hd=96, mix=9),
        # a pool half of whose sequences have ended
        dict(name="compact_180", op="compact", n=180, pages=400, nseq=64, ld=128, layers=28, KV=8, hd=128, mix=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["attend", "attend", "attend", "append", "fork", "compact"])
        mix, hd = rng.randrange(1 << 30), GROUP * rng.choice([1, 2, 2, 3, 4, 4, 4, 5, 6, 7, 8])
        if op == "attend":
            KV = rng.choice([1, 2, 3, 4, 4, 8, 8, 16])
            H = KV * rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16])
            if rng.random() < 0.6:
                nseq, rows, max_len = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 4, 5]), _log(rng, 8, 131072)
            else:
                nseq, rows, max_len = _log(rng, 1, 12), _log(rng, 6, 2048), _log(rng, 8, 8192)
            rows = min(rows, max_len)
            window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
            case = dict(op=op, nseq=nseq, rows=rows, max_len=max_len, H=H, KV=KV, hd=hd, window=window,
                        ragged=rng.random() < 0.7, mix=mix)
        elif op == "append":
            max_len = _log(rng, 1, 8192)
            case = dict(op=op, nseq=_log(rng, 1, 96), rows=min(max_len, _log(rng, 1, 4096)), max_len=max_len,
                        KV=rng.choice([1, 2, 3, 4, 8, 16]), hd=hd, ragged=rng.random() < 0.7, mix=mix)
        elif op == "fork":
            nsrc = _log(rng, 1, 16)
            case = dict(op=op, n=nsrc * rng.randint(1, 4), nsrc=nsrc, max_len=_log(rng, 1, 2000), layers=rng.randint(1, 32),
                        KV=rng.choice([1, 2, 3, 4, 8]), hd=hd, mix=mix)
        else:
            n = _log(rng, 1, 180)
            case = dict(op=op, n=n, pages=2 * n + rng.randint(1, 60), nseq=rng.randint(1, 64), ld=rng.randint(1, 128),
                        layers=rng.randint(1, 32), KV=rng.choice([1, 2, 3, 4, 8]), hd=hd, mix=mix)
        w = work(case)
        # (the pool of a fork or a compaction is an output too: it stays below the largest listed one)
        pool = case.get("pages", 0) * _page_bytes(case) if op == "compact" else 0
        if op == "fork":
            pool = _fork_pages(case) * _page_bytes(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and pool <= 830 << 20:
            return case


def _page_bytes(case):
    return case.get("layers", 1) * case["KV"] * 72 * case["hd"]


def _lens(case):
    """(rows, len) of every sequence, from the case alone."""
    r = random.Random(case["mix"])
    out = []
    for s in range(case["nseq"]):
        n, L = case["rows"], case["max_len"]
        if case["ragged"] and s > 0:
            n = 1 if r.random() < 0.34 else r.randint(max(1, n // 4), n)
            L = r.randint(max(n, L // 8), L)
        out.append((n, L))
    return out


def _first_page(case, n, L):
    """Pages wholly in front of the window have been freed."""
    w = case.get("window", 0)
    return max(0, L - n - w + 1) // PAGE if w else 0


def _visible(case, n, L):
    """(positions that some row sees, sum over rows of positions seen)"""
    w = case.get("window", 0) or L
    lo = max(0, L - n - w + 1)
    return L - lo, sum(min(p + 1, w) for p in range(L - n, L))


def work(case):
    if case["op"] == "attend":
        b = f = 0
        for n, L in _lens(case):
            seen, pairs = _visible(case, n, L)
            b += seen * case["KV"] * case["hd"] * 9 // 8 + 2 * n * case["H"] * case["hd"] * 4 + 4 * ((seen + PAGE - 1) // PAGE) + 8
            f += 4 * case["H"] * case["hd"] * pairs
        return {"bytes": b, "flops": f}
    if case["op"] == "append":              # rows in as f32 and out again as the values held; the 4-bit rows written and read
        n = sum(n for n, _ in _lens(case)) * case["KV"] * case["hd"]
        return {"bytes": n * (8 + 8) + 2 * n * 9 // 8, "flops": 8 * n}
    if case["op"] == "fork":
        tails = sum(1 for L in _fork_lens(case) if L % PAGE)
        return {"bytes": 2 * tails * _page_bytes(case) + 2 * 4 * sum((L + PAGE - 1) // PAGE for L in _fork_lens(case)), "flops": 0}
    return {"bytes": 2 * case["n"] * _page_bytes(case) + 2 * 4 * case["nseq"] * case["ld"], "flops": 0}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _rows_like(g, shape, outliers):
    """Projections as the path meets them: normal, keys with a few channels several times the others."""
    x = torch.randn(shape, generator=g, device=DEV)
    return x * (1.0 + 3.0 * (outliers < 0.03)) if outliers is not None else x


def _batch(case, g):
    """Lengths, row offsets and a page table over a shuffled pool."""
    lens = _lens(case)
    need = [(L + PAGE - 1) // PAGE for _, L in lens]
    ld, pages = max(need) + 1, sum(need) + 3
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["nseq"], ld), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, (n, L) in enumerate(lens):
        f = _first_page(case, n, L)
        table[s, f:need[s]] = perm[at + f:at + need[s]]
        at += need[s]
    row0 = [0]
    for n, _ in lens:
        row0.append(row0[-1] + n)
    return dict(lens=lens, row0=row0, row0_dev=_ints(row0), len_dev=_ints([L for _, L in lens]), table=table, ld=ld, pages=pages)


def _kv(case, g, n, chan):
    return (_rows_like(g, (n, case["KV"], case["hd"]), chan), _rows_like(g, (n, case["KV"], case["hd"]), None))


def _attend_inputs(case, seed):
    g = _gen(seed)
    b = _batch(case, g)
    chan = torch.rand((case["KV"], case["hd"]), generator=g, device=DEV)
    b["q"] = torch.randn((b["row0"][-1], case["H"], case["hd"]), generator=g, device=DEV)
    # the rows of each sequence from its first kept page on (what was freed before the window is not made)
    b["kv"] = lambda s: _kv(case, _gen(seed * 1009 + 17 * s + 1), b["lens"][s][1] - PAGE * _first_page(case, *b["lens"][s]), chan)
    return b


def _append_inputs(case, seed):
    g = _gen(seed)
    b = _batch(case, g)
    chan = torch.rand((case["KV"], case["hd"]), generator=g, device=DEV)
    b["k"], b["v"] = _kv(case, g, b["row0"][-1], chan)
    return b


def _fork_lens(case):
    r = random.Random(case["mix"])
    src = [r.randint(max(1, case["max_len"] // 2), case["max_len"]) for _ in range(case["nsrc"])]
    return [src[i % case["nsrc"]] for i in range(case["n"])]


def _fork_pages(case):
    return sum((L + PAGE - 1) // PAGE for L in _fork_lens(case)[:case["nsrc"]]) + case["n"] + 2


def _fork_inputs(case, seed):
    g = _gen(seed)
    n, nsrc, lens = case["n"], case["nsrc"], _fork_lens(case)
    pages, rows = _fork_pages(case), nsrc + n
    ld = (case["max_len"] + PAGE - 1) // PAGE + 1
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((rows, ld), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s in range(nsrc):
        k = (lens[s] + PAGE - 1) // PAGE
        table[s, :k] = perm[at:at + k]
        at += k
    new = perm[at:at + n].clone()
    for i in range(n):
        if lens[i] % PAGE == 0:
            new[i] = -1                                     # a sequence that ends on a page has no tail to copy
    length = _ints(lens[:nsrc] + [0] * n)
    mem = torch.randint(-1 << 31, 1 << 31, (pages, _page_bytes(case) // 4), generator=g, device=DEV, dtype=torch.int32)
    return dict(mem=mem, pages=pages, table=table, len_dev=length, new=new, src=_ints([i % nsrc for i in range(n)]),
                dst=_ints([nsrc + i for i in range(n)]), rows=rows, ld=ld, lens=lens)


def _compact_inputs(case, seed):
    g = _gen(seed)
    r = random.Random(case["mix"])
    pages, n = case["pages"], case["n"]
    # n holes below, n live pages above the boundary `live`
    live = r.randint(n, pages - n)
    dst = sorted(r.sample(range(live), n))
    src = sorted(r.sample(range(live, pages), n))
    ids = sorted(set(range(live)) - set(dst)) + src
    pick = torch.randint(0, len(ids), (case["nseq"], case["ld"]), generator=g, device=DEV)
    table = _ints(ids)[pick]
    used = torch.randint(0, case["ld"] + 1, (case["nseq"], 1), generator=g, device=DEV)
    table = torch.where(torch.arange(case["ld"], device=DEV)[None] < used, table, torch.full_like(table, -1))
    mem = torch.randint(-1 << 31, 1 << 31, (pages, _page_bytes(case) // 4), generator=g, device=DEV, dtype=torch.int32)
    return dict(mem=mem, pages=pages, table=table, out=torch.empty_like(table), src=_ints(src), dst=_ints(dst))


_INPUTS = {"attend": _attend_inputs, "append": _append_inputs, "fork": _fork_inputs, "compact": _compact_inputs}


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _quant(x):
    """x [..][hd] f32 -> (codes 0..15 uint8 of the same shape, steps f16 [..][hd / 32])"""
    v = x.reshape(*x.shape[:-1], -1, GROUP)
    a = v.abs()
    m = a.max(-1, keepdim=True).values
    first = (a == m).to(torch.uint8).argmax(-1, keepdim=True)
    big = torch.gather(v, -1, first)
    other = torch.where((v > 0) != (big > 0), a, torch.zeros_like(a)).max(-1, keepdim=True).values
    # (a true division: dividing by a Python number multiplies by its reciprocal on the GPU, another rounding)
    step = torch.maximum(big.abs() / 8, other / torch.full_like(other, 7.0)).clamp(max=65504.0)
    d = torch.where(big > 0, -step, step).to(torch.float16)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    d = torch.where(bad, torch.full_like(d, math.nan), d)
    df = d.float()
    code = torch.where((df == 0) | bad, torch.zeros_like(v), torch.round(v / df)).clamp(-8, 7)
    return (code + 8).to(torch.uint8).reshape(x.shape), d.squeeze(-1)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(packed, steps):
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], -1).float() - 8
    v = code.reshape(*steps.shape, GROUP) * steps.float()[..., None]
    return v.reshape(code.shape)


def _plain_pool(case, pages):
    KV, hd = case["KV"], case["hd"]
    return dict(kc=torch.zeros((pages, KV, PAGE, hd // 2), dtype=torch.uint8, device=DEV),
                ks=torch.zeros((pages, KV, PAGE, hd // GROUP), dtype=torch.float16, device=DEV),
                vc=torch.zeros((pages, KV, PAGE, hd // 2), dtype=torch.uint8, device=DEV),
                vs=torch.zeros((pages, KV, PAGE, hd // GROUP), dtype=torch.float16, device=DEV))


def _plain_store(pool, k, v, page, slot):
    """rows k, v [n][KV][hd] to positions `slot` of pages `page` (both [n])"""
    for x, c, s in ((k, "kc", "ks"), (v, "vc", "vs")):
        code, step = _quant(x)
        pool[c][page, :, slot] = _pack(code)
        pool[s][page, :, slot] = step


def _plain_rows(pool, page, slot):
    return (_values(pool["kc"][page, :, slot], pool["ks"][page, :, slot]),
            _values(pool["vc"][page, :, slot], pool["vs"][page, :, slot]))


def _plain_attend(st):
    case, out = st["case"], []
    H, KV, hd, w = case["H"], case["KV"], case["hd"], case["window"]
    G = H // KV
    for s, (n, L) in enumerate(st["lens"]):
        lo = PAGE * _first_page(case, n, L)
        pos = torch.arange(lo, L, device=DEV)
        page = st["table"][s][pos // PAGE].long()
        k, v = _plain_rows(st["pool"], page, pos % PAGE)                    # [T][KV][hd]
        q = st["q"][st["row0"][s]:st["row0"][s] + n]
        qpos = torch.arange(L - n, L, device=DEV)
        hide = pos[None, :] > qpos[:, None]
        if w:
            hide |= pos[None, :] <= qpos[:, None] - w
        ctx = torch.empty((n, H, hd), device=DEV)
        for h in range(KV):
            sc = (q[:, h * G:(h + 1) * G].reshape(n * G, hd) @ k[:, h].t()).reshape(n, G, -1) * (1.0 / math.sqrt(hd))
            sc = sc.masked_fill(hide[:, None], -math.inf)
            p = torch.exp(sc - sc.max(-1, keepdim=True).values)
            o = (p.reshape(n * G, -1) @ v[:, h]).reshape(n, G, hd) / p.sum(-1, keepdim=True)
            ctx[:, h * G:(h + 1) * G] = o
        out.append(ctx)
    return torch.cat(out).reshape(st["row0"][-1], H * hd)


def _plain_append(st):
    _plain_store(st["pool"], st["k"], st["v"], st["page"], st["slot"])
    return _plain_rows(st["pool"], st["page"], st["slot"])


def _plain_fork(st):
    mem, table, length = st["mem"], st["table"], st["len_dev"]
    for i, L in enumerate(st["lens"]):
        s, d = i % st["case"]["nsrc"], st["case"]["nsrc"] + i
        full = L // PAGE
        table[d] = -1
        table[d, :full] = table[s, :full]
        length[d] = length[s]
    tail = [i for i, L in enumerate(st["lens"]) if L % PAGE]
    if tail:
        i = torch.tensor(tail, device=DEV)
        full = torch.tensor([st["lens"][j] // PAGE for j in tail], device=DEV)
        table[st["dst"][i].long(), full] = st["new"][i]
        mem[st["new"][i].long()] = mem[table[st["src"][i].long(), full].long()]
    return mem, table, length


def _plain_compact(st):
    st["mem"][st["dst"].long()] = st["mem"][st["src"].long()]
    name = torch.arange(-1, st["pages"], device=DEV, dtype=torch.int32)     # name[id + 1]; -1 stays -1
    name[st["src"].long() + 1] = st["dst"]
    st["out"].copy_(name[st["table"].long() + 1])
    return st["mem"], st["out"]


# ---- the library's calls ----------------------------------------------------------------------------------------------
def _stream():
    import moty_b200 as mb
    return mb.stream_handle(torch.cuda.current_stream())


def _own_pool(case, pages, mem=None):
    """The handle over memory that the program allocated (the pages' bytes are the program's own tensor)."""
    import moty_b200 as mb
    mb.init([torch.cuda.current_device()])
    layers = case.get("layers", 1)
    if mem is None:
        mem = torch.zeros((pages, mb.Kv4.page_bytes(layers, case["KV"], case["hd"]) // 4), dtype=torch.int32, device=DEV)
    return mb.Kv4(layers, case["KV"], case["hd"], pages, device=torch.cuda.current_device(), mem_ptr=mem.data_ptr()), mem


def _own_batch(st):
    import moty_b200 as mb
    return mb.Kv4Batch(len(st["lens"]), st["row0"][-1], st["row0_dev"].data_ptr(), st["len_dev"].data_ptr(), st["table"].data_ptr(),
                       st["ld"], max_rows=max(n for n, _ in st["lens"]), max_len=max(L for _, L in st["lens"]))


# ---- prepare, run -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    st["case"] = case
    if case["op"] == "attend":
        if own:
            import moty_b200 as mb
            st["kv4"], st["mem"] = _own_pool(case, st["pages"])
            st["ctx"] = torch.empty((st["row0"][-1], case["H"] * case["hd"]), device=DEV)
            st["batch"] = _own_batch(st)
        else:
            st["pool"] = _plain_pool(case, st["pages"])
        for s, (n, L) in enumerate(st["lens"]):
            k, v = st["kv"](s)
            f = _first_page(case, n, L)
            if own:
                row0, ln = _ints([0, k.shape[0]]), _ints([L])
                one = mb.Kv4Batch(1, k.shape[0], row0.data_ptr(), ln.data_ptr(), st["table"][s].data_ptr(), st["ld"],
                                  max_rows=k.shape[0], max_len=L)
                st["kv4"].append_dev(0, k.data_ptr(), v.data_ptr(), one, stream=_stream())
                torch.cuda.current_stream().synchronize()
            else:
                pos = torch.arange(PAGE * f, L, device=DEV)
                _plain_store(st["pool"], k, v, st["table"][s][pos // PAGE].long(), pos % PAGE)
        del st["kv"]
    elif case["op"] == "append":
        if own:
            st["kv4"], st["mem"] = _own_pool(case, st["pages"])
            st["batch"] = _own_batch(st)
            st["k_held"], st["v_held"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        else:
            st["pool"] = _plain_pool(case, st["pages"])
            pos = torch.cat([torch.arange(L - n, L, device=DEV) for n, L in st["lens"]])
            seq = torch.cat([torch.full((n,), s, device=DEV) for s, (n, _) in enumerate(st["lens"])])
            st["page"], st["slot"] = st["table"][seq, pos // PAGE].long(), pos % PAGE
    elif own:
        st["kv4"], _ = _own_pool(case, st["pages"], st["mem"])
    return st


def run(st):
    case = st["case"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact}[case["op"]](st)
    kv, sh = st["kv4"], _stream()
    if case["op"] == "attend":
        kv.attend_dev(0, st["ctx"].data_ptr(), st["q"].data_ptr(), case["H"], st["batch"], window=case["window"], stream=sh)
        return st["ctx"]
    if case["op"] == "append":
        kv.append_dev(0, st["k"].data_ptr(), st["v"].data_ptr(), st["batch"], stream=sh)
        kv.fetch_dev(0, st["k_held"].data_ptr(), st["v_held"].data_ptr(), st["batch"], stream=sh)
        return st["k_held"], st["v_held"]
    if case["op"] == "fork":
        kv.fork_dev(case["n"], st["src"].data_ptr(), st["dst"].data_ptr(), st["new"].data_ptr(), st["rows"], st["len_dev"].data_ptr(),
                    st["table"].data_ptr(), st["ld"], stream=sh)
        return st["mem"], st["table"], st["len_dev"]
    kv.compact_dev(case["n"], st["src"].data_ptr(), st["dst"].data_ptr(), st["table"].numel(), st["table"].data_ptr(),
                   st["out"].data_ptr(), stream=sh)
    return st["mem"], st["out"]


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _held64(x):
    """The values the cache holds for rows x, in f64 (the step's two roundings, f32 and f16, are part of the format)."""
    t = x.double().unflatten(-1, (-1, GROUP))
    hi, lo = t.amax(-1), t.amin(-1)
    # the side that reaches farther gets the code -8; on equal reach the side whose value comes first
    pos_first = (t == hi[..., None]).int().argmax(-1) < (t == lo[..., None]).int().argmax(-1)
    pos_big = (hi > -lo) | ((hi == -lo) & pos_first)
    far = torch.where(pos_big, hi, -lo).clamp(min=0)
    near = torch.where(pos_big, -lo, hi).clamp(min=0)
    step = torch.maximum((far / 8).float(), (near / 7).float())
    d = (torch.where(pos_big, -1.0, 1.0) * step.clamp(max=65504.0)).half().double()[..., None]
    code = torch.where(d == 0, torch.zeros_like(t), (t / d).round().clamp(-8, 7))
    return (code * d).flatten(-2)


def exact(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    if case["op"] == "append":
        return _held64(st["k"]), _held64(st["v"])
    if case["op"] == "fork":
        table, length, mem = st["table"].cpu(), st["len_dev"].cpu(), st["mem"]
        for src, dst, new in zip(st["src"].tolist(), st["dst"].tolist(), st["new"].tolist()):
            L = int(length[src])
            row = table[src, :L // PAGE].tolist()
            if L % PAGE:
                mem[new] = mem[int(table[src, L // PAGE])]
                row.append(new)
            table[dst] = torch.tensor(row + [-1] * (table.shape[1] - len(row)), dtype=torch.int32)
            length[dst] = L
        return mem, table.to(DEV), length.to(DEV)
    if case["op"] == "compact":
        moved = dict(zip(st["src"].tolist(), st["dst"].tolist()))
        for a, b in moved.items():
            st["mem"][b] = st["mem"][a]
        return st["mem"], _ints([[moved.get(p, p) for p in row] for row in st["table"].tolist()])
    H, KV, hd, w = case["H"], case["KV"], case["hd"], case["window"]
    out = torch.empty((st["row0"][-1], KV, H // KV, hd), dtype=torch.float64, device=DEV)
    for s, (n, L) in enumerate(st["lens"]):
        k, v = st["kv"](s)
        k, v, lo = _held64(k), _held64(v), L - k.shape[0]
        for at in range(0, n, 1024):                        # a block of rows at a time
            r0, r1 = st["row0"][s] + at, st["row0"][s] + min(n, at + 1024)
            q = st["q"][r0:r1].double().unflatten(1, (KV, H // KV))
            here = torch.arange(L - n + at, L - n + at + (r1 - r0), device=DEV)[:, None]
            there = torch.arange(lo, L, device=DEV)[None]
            seen = there <= here
            if w:
                seen &= there > here - w
            for h in range(KV):
                z = torch.einsum("ngd,td->ngt", q[:, h], k[:, h]) / math.sqrt(hd)
                z = torch.where(seen[:, None], z, torch.full_like(z, -math.inf))
                out[r0:r1, h] = torch.einsum("ngt,td->ngd", torch.softmax(z, -1), v[:, h])
    return out.reshape(-1, H * hd)
