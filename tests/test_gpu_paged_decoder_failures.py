"""GPU: PagedDecoder when a call fails on the host -- an allocation, a launch, the kernels' status -- and what forks share.  The
failures are raised by the test in place of the real call; nothing faults on the GPU."""
import numpy as np
import pytest

from test_gpu_paged_decoder import _model

pytestmark = pytest.mark.gpu

H, KV, HD, V = 4, 2, 32, 300


def make(gpu, **kw):
    from moty_b200.decoder import PagedDecoder
    W, layers, head = _model(gpu, np.random.default_rng(4), H, KV, HD, 128, 256, V, 2, True)
    return PagedDecoder(layers, head, W["final_norm"], H, KV, HD, **{**dict(pages=10, max_seqs=5, max_pages=4), **kw})


def state(dec):
    return dec.table.tolist(), dec.lens.tolist(), dec.used.tolist(), dec.kv.free_pages()


class Failure(Exception):
    pass


def fail(*a, **k):
    raise Failure


def failing(monkeypatch, dec, what):
    """`what` of the decoder raises: as a method, or (after:) once the real one has been called."""
    if what.startswith("after:"):
        name = what[6:]
        real = getattr(dec, name)

        def call(*a, **k):
            real(*a, **k)
            raise Failure
        monkeypatch.setattr(dec, name, call)
    else:
        monkeypatch.setattr(dec, what, fail)


@pytest.mark.parametrize("what", ["_embed_rows", "_layers_paged", "after:_layers_paged", "_head", "after:_head", "_check_kernels"])
@pytest.mark.parametrize("call", ["run", "greedy"])
def test_a_step_that_fails_changes_nothing(gpu, monkeypatch, call, what):
    rng = np.random.default_rng(1)
    prompt, more = rng.integers(0, V, 60), rng.integers(0, V, 80)
    good = make(gpu)
    a = good.new()
    good.run([(a, prompt)])
    want, want_lg = good.run([(a, more)], want_logits=True)
    dec = make(gpu)
    s, other = dec.new(), dec.new()
    tok = dec.run([(s, prompt)])
    dec.run([(other, prompt[:5])])
    before = state(dec)
    for _ in range(2):
        with monkeypatch.context() as m:
            failing(m, dec, what)
            with pytest.raises(Failure):
                dec.run([(s, more), (other, [1])]) if call == "run" else dec.greedy([s, other], [int(tok[0]), 1], 70)
        assert state(dec) == before
    out, lg = dec.run([(s, more)], want_logits=True)
    assert out[0] == want[0] and np.array_equal(lg, want_lg)
    good.close(); dec.close()


@pytest.mark.parametrize("tokens", [70, 64])                 # with a partial last page and without
@pytest.mark.parametrize("what", ["fork_dev", "retain", "_check_kernels"])
def test_a_fork_that_fails_changes_nothing(gpu, monkeypatch, what, tokens):
    dec = make(gpu)
    s = dec.new()
    dec.run([(s, np.arange(tokens))])
    before = state(dec)
    for _ in range(2):
        with monkeypatch.context() as m:
            m.setattr(dec if what == "_check_kernels" else dec.kv, what, fail)
            with pytest.raises(Failure):
                dec.fork(s, 2)
        assert state(dec) == before
    assert dec.new() == 1                                    # a sequence of nothing, as before
    dec.end(1)
    f = dec.fork(s, 2)
    out, lg = dec.run([(x, [7]) for x in [s] + f], want_logits=True)
    assert np.array_equal(lg[0], lg[1]) and np.array_equal(lg[0], lg[2])
    for x in [s] + f:
        dec.end(x)
    assert dec.kv.free_pages() == 10
    dec.close()


@pytest.mark.parametrize("what", ["to", "plan", "move", "_check_kernels"])
def test_a_compaction_that_fails(gpu, monkeypatch, what):
    """For want of memory, or of a plan: nothing has changed, and it can be asked again.  In the moves: every call is refused."""
    dec = make(gpu)
    a, b = dec.new(), dec.new()
    dec.run([(a, np.arange(70)), (b, np.arange(100))])
    dec.end(a)
    before = state(dec)
    with monkeypatch.context() as m:
        if what == "to":
            m.setattr(dec, "dev", "nowhere")                 # (no tensor can be made there)
        elif what == "_check_kernels":
            m.setattr(dec, what, fail)
        else:
            m.setattr(dec.kv, {"plan": "compact_plan", "move": "compact_dev"}[what], fail)
        with pytest.raises((Failure, RuntimeError)):
            dec.compact()
    assert state(dec)[1:] == before[1:]
    if what in ("to", "plan"):
        assert dec.table.tolist() == before[0]
        want = make(gpu)
        x = want.new(); want.run([(x, np.arange(100))])
        assert dec.compact() > 0 and sorted(dec.table[dec.table >= 0].tolist()) == [0, 1]
        assert np.array_equal(dec.run([(b, [3])], want_logits=True)[1], want.run([(x, [3])], want_logits=True)[1])
        want.close()
    else:
        for call in (lambda: dec.run([(b, [3])]), lambda: dec.fork(b), lambda: dec.greedy([b], [3], 2), lambda: dec.end(b), dec.new, dec.compact):
            with pytest.raises(gpu.MotyCudaError, match="compaction"):
                call()
    dec.close()


def held(gpu, dec, sid):
    """The key and value rows that a sequence holds, every layer."""
    import torch
    n = int(dec.lens[sid])
    d = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")
    row0, ln, tab = d([0, n]), d([n]), d(dec.table[sid])
    b = gpu.Kv4Batch(1, n, row0.data_ptr(), ln.data_ptr(), tab.data_ptr(), dec.max_pages)
    out = []
    for layer in range(len(dec.layers)):
        k, v = (torch.full((n, KV * HD), 9.0, device="cuda") for _ in range(2))
        dec.kv.fetch_dev(layer, k.data_ptr(), v.data_ptr(), b, stream=gpu.stream_handle(torch.cuda.current_stream()))
        out.append(np.stack([k.cpu().numpy(), v.cpu().numpy()]))
    return np.stack(out)


@pytest.mark.parametrize("tokens", [70, 64])
def test_what_forks_append_is_their_own(gpu, tokens):
    """Forks that go on differently: full pages shared, last pages each one's own, and every sequence's earlier rows byte for byte
    what they were."""
    dec = make(gpu)
    s = dec.new()
    dec.run([(s, np.arange(tokens) * 3 % V)])
    before = held(gpu, dec, s)
    forks = dec.fork(s, 2)
    for step in range(3):
        dec.run([(x, [(50 * i + step) % V]) for i, x in enumerate([s] + forks)])
    full = tokens // 64
    last = [int(dec.table[x, full]) for x in [s] + forks]
    assert len(set(last)) == 3 and min(last) >= 0
    for x in forks:
        assert dec.table[x, :full].tolist() == dec.table[s, :full].tolist()
    rows = [held(gpu, dec, x) for x in [s] + forks]
    for r in rows:
        assert r[:, :, :tokens].tobytes() == before.tobytes()
    assert not np.array_equal(rows[0][:, :, tokens:], rows[1][:, :, tokens:]) and not np.array_equal(rows[1][:, :, tokens:], rows[2][:, :, tokens:])
    dec.close()


def test_greedy_leaves_the_scratch_frozen_for_others(gpu):
    """A captured step of another decoder holds the library's scratch addresses: after a greedy call beside it the scratch still
    does not move."""
    L = gpu.lib()
    dec = make(gpu)
    s = dec.new()
    tok = dec.run([(s, np.arange(70))])
    dec.greedy([s], tok, 2)                                  # (the scratch it needs is there)
    W = gpu.Mat.i8(np.zeros((64, 4096), np.int8), np.ones(64, np.float32))
    gpu._ck(L.moty_cuda_scratch_freeze(0, 1))
    try:
        dec.greedy([s], [1], 2)
        with pytest.raises(gpu.MotyCudaError, match="frozen"):
            gpu.mat_apply(W, np.zeros((60000, 4096), np.float32))
    finally:
        gpu._ck(L.moty_cuda_scratch_freeze(0, 0))
    dec.greedy([s], [1], 2)
    dec.close()


def test_a_decoder_that_closes_leaves_the_scratch_frozen_for_others(gpu):
    """Two decoders with captured steps: the scratch moves again when the last of them has let go."""
    from moty_b200.decoder import DenseDecoder
    W, layers, head = _model(gpu, np.random.default_rng(4), H, KV, HD, 128, 256, V, 2, True)
    one, two = (DenseDecoder(layers, head, W["final_norm"], H, KV, HD, 64) for _ in range(2))
    want = one.greedy_graph(3, 0, 4)
    assert two.greedy_graph(3, 0, 4) == want
    two.close()
    big = gpu.Mat.i8(np.zeros((64, 4096), np.int8), np.ones(64, np.float32))
    x = np.zeros((60000, 4096), np.float32)
    with pytest.raises(gpu.MotyCudaError, match="frozen"):
        gpu.mat_apply(big, x)
    assert one.greedy_graph(3, 0, 4) == want
    one.close()
    assert DenseDecoder._holders[0] == 0
