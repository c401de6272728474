"""A dense decoder step on one GPU, composed from the library's device entries the way the reference's
``qwen`` engine composes its CPU functions (engines/qwen.c:681-740, ``step``): embedding rows, then per
layer RMS norm -> q/k/v projections -> attention core -> o projection -> residual add -> RMS norm ->
SwiGLU FFN -> residual add, then the final norm of the last token, the (tied) lm_head and the greedy
pick.  Activations stay on the device; only token ids go in and one id (or the logits) comes out.

This is host-side glue for tests and for the decode rows of ``bench.py``; the arithmetic is in the C-ABI
entries it calls (``moty_cuda_mat_apply_dev``, ``moty_cuda_attn_core_dev``, ``moty_cuda_ffn_dev``,
``moty_cuda_rmsnorm_dev``, ``moty_cuda_add_dev``, ``moty_cuda_embed_rows_dev``, ``moty_cuda_head_argmax_dev``).
"""
from __future__ import annotations

import contextlib
import ctypes as C

import numpy as np

from . import Attn, Kv4, Kv4Batch, Mat, MotyCudaError, lib, stream_handle, ACT_GELU_TANH, ACT_SILU


def _ck(rc):
    if rc != 0:
        raise MotyCudaError(f"libmoty_cuda error {rc}: {lib().moty_cuda_last_error().decode()}")


class DenseLayer:
    """One layer's weights: int8 matrices (q, k, v, o, gate, up, down) and f32 norm gains."""

    def __init__(self, q, k, v, o, gate, up, down, in_ln, post_ln, qn=None, kn=None, qkv=None, moe=None, norm_topk=1):
        self.q, self.k, self.v, self.o, self.gate, self.up, self.down = q, k, v, o, gate, up, down
        self.in_ln, self.post_ln, self.qn, self.kn = in_ln, post_ln, qn, kn
        # optional: the rows of q, k and v in one matrix (the reference's fused [q|k|v], nn/attn.h:24): one product
        # per decode token instead of three; per-row quantization makes the concatenation exact
        self.qkv = qkv
        # optional: a routed layer (moty_b200.Moe with its router set) in place of the dense FFN, combined per token in
        # selection order as engines/olmoe.c:219-244 does; gate/up/down may then be None
        self.moe, self.norm_topk = moe, norm_topk


class DenseDecoder:
    """``layers``: list of DenseLayer (matrices as ``moty_b200.Mat``, gains as numpy f32); ``head``: the lm_head
    ``Mat`` (MOTY_WF_I8 [vocab][D]; with tied embeddings it is also the embedding table); ``final_norm`` [D]."""

    def __init__(self, layers, head: Mat, final_norm, n_heads, n_kv_heads, head_dim, max_t, theta=1e6, eps=1e-6,
                 rot=None, kv8=False, device=0, max_S=64, fold_addnorm=None, fold_ffn=False):
        import torch
        self.torch = torch
        self.dev = torch.device(f"cuda:{device}")
        self.layers, self.head = layers, head
        self.H, self.KV, self.hd, self.eps, self.max_t = n_heads, n_kv_heads, head_dim, float(eps), max_t
        self.D = head.I
        # fold the add+norm in front of a layer's [q|k|v] product into that launch (one token): measured a gain at hidden
        # 1024 (1391 -> 1428 tok/s replayed) and 2048 once every launch of the layer was chained to the next.  The same
        # fold in front of the dense FFN block (fold_ffn) is built and bit-identical but measured a loss (1428 -> 1398):
        # the ~600 CTAs of the gate/up launch each redo the row, where the separate one-CTA launch is nearly free
        self.fold_addnorm = True if fold_addnorm is None else bool(fold_addnorm)
        self.fold_ffn = bool(fold_ffn)
        f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(self.dev)
        self.final_norm = f(final_norm)
        self.ln = [(f(l.in_ln), f(l.post_ln)) for l in layers]
        self.attn = [Attn(n_heads, n_kv_heads, head_dim, max_t, theta=theta, eps=eps, rot=rot, qn=l.qn, kn=l.kn, kv8=kv8,
                          device=device) for l in layers]
        self.stream = torch.cuda.Stream(device=self.dev)
        self._alloc(max_S)

    def _alloc(self, S):
        t, dev = self.torch, self.dev
        qw, kw = self.H * self.hd, self.KV * self.hd
        e = lambda *shape: t.empty(shape, device=dev, dtype=t.float32)
        self._drop_graph()                       # a captured step holds the addresses of the buffers replaced below
        self.cap = 0                             # until all of them are there: a failed allocation must not leave small ones for S rows
        self.x, self.nrm, self.tmp = e(S, self.D), e(S, self.D), e(S, self.D)
        self.x_alt = e(1, self.D)
        self.qb, self.kb, self.vb, self.ctx = e(S, qw), e(S, kw), e(S, kw), e(S, qw)
        self.qkvb = e(1, qw + 2 * kw)
        self.ids = t.empty((S,), device=dev, dtype=t.int32)
        self.out_id = t.empty((1,), device=dev, dtype=t.int32)
        self.logits = e(1, self.head.O)
        self.cap = S

    def _drop_graph(self):
        """Forget the captured decode step and, unless another decoder holds one, let the library's scratch grow again."""
        if getattr(self, "_graph", None) is not None:
            self._graph = None
            self._hold_scratch(-1)

    _holders = {}                                # device -> captured steps that hold the addresses of its scratch

    def _hold_scratch(self, n):
        d = self.dev.index or 0
        held = self._holders[d] = self._holders.get(d, 0) + n
        if held == (1 if n > 0 else 0):
            _ck(lib().moty_cuda_scratch_freeze(d, int(n > 0)))

    def _check_kernels(self):
        """After a stream synchronisation: did a bounded wait inside a kernel run out (incomplete results)?"""
        _ck(lib().moty_cuda_kernel_status(self.dev.index or 0, C.c_void_p(stream_handle(self.stream))))

    def step(self, ids, pos_base, want_logits=False):
        """Tokens ``ids`` at positions pos_base.. : returns the greedy next token after the last of them
        (and the last token's logits when asked)."""
        t, L = self.torch, lib()
        ids = np.ascontiguousarray(ids, np.int32).ravel()
        S = ids.size
        if S > getattr(self, "_max_S", 0):
            self._drop_graph()                   # a larger batch than any before may grow the library's scratch
            self._max_S = S
        if S > self.cap:
            self._alloc(S)
        if pos_base + S > self.max_t:
            raise MotyCudaError(f"positions {pos_base}..{pos_base + S} exceed the cache of {self.max_t}")
        D = self.D
        p = lambda ten: C.c_void_p(ten.data_ptr())
        with t.cuda.stream(self.stream):
            sh = C.c_void_p(stream_handle(self.stream))
            self.ids[:S].copy_(t.from_numpy(ids), non_blocking=True)
            _ck(L.moty_cuda_embed_rows_dev(self.head.h, p(self.x), p(self.ids), S, C.c_float(1.0), sh))
            x = self._layers(S, pos_base, None, sh)
            last = x[S - 1:S]
            _ck(L.moty_cuda_rmsnorm_dev(p(self.nrm), p(last), p(self.final_norm), 1, D, C.c_float(self.eps), sh))
            _ck(L.moty_cuda_head_argmax_dev(self.head.h, p(self.nrm), 1, p(self.out_id), p(self.logits), sh))
            tok = int(self.out_id.cpu()[0])          # waits for the stream
            self._check_kernels()
            if want_logits:
                return tok, self.logits.cpu().numpy()[0]
        return tok

    def _layers(self, S, pos_base, pos_dev, sh):
        """The layers of engines/qwen.c:696-712 on self.x [S][D].  A residual add and the norm that follows it are one
        launch (same results); with S = 1 and a fused matrix the three projections are one product, and the add+norm in
        front of that product and in front of a dense FFN block ride inside those launches (same bits; the sum goes to
        the other of two residual buffers)."""
        L, D, eps = lib(), self.D, C.c_float(self.eps)
        p = lambda ten: C.c_void_p(ten.data_ptr())
        qw, kw = self.H * self.hd, self.KV * self.hd
        nl = len(self.layers)
        x, x_alt = self.x, self.x_alt
        one = self.fold_addnorm and S == 1
        fold_qkv = [one and l.qkv is not None and bool(L.moty_cuda_mat_addnorm_supported(l.qkv.h)) for l in self.layers]
        fold_ffn = [self.fold_ffn and S == 1 and l.moe is None and bool(L.moty_cuda_ffn_resnorm_supported(l.gate.h, l.up.h))
                    for l in self.layers]
        pending = False                          # self.tmp holds a block output that has not been added to x yet
        _ck(L.moty_cuda_rmsnorm_dev(p(self.nrm), p(x), p(self.ln[0][0]), S, D, eps, sh))
        for i, (l, (in_ln, post_ln), a) in enumerate(zip(self.layers, self.ln, self.attn)):
            if S == 1 and l.qkv is not None:
                if pending:
                    _ck(L.moty_cuda_mat_apply_resnorm_dev(l.qkv.h, p(self.qkvb), p(x), p(self.tmp), None, p(x_alt), p(in_ln), eps, sh))
                    x, x_alt = x_alt, x
                    pending = False
                else:
                    _ck(L.moty_cuda_mat_apply_dev(l.qkv.h, p(self.qkvb), p(self.nrm), 1, sh))
                base = self.qkvb.data_ptr()
                qp, kp, vp = C.c_void_p(base), C.c_void_p(base + 4 * qw), C.c_void_p(base + 4 * (qw + kw))
            else:
                _ck(L.moty_cuda_mat_apply_dev(l.q.h, p(self.qb), p(self.nrm), S, sh))
                _ck(L.moty_cuda_mat_apply_dev(l.k.h, p(self.kb), p(self.nrm), S, sh))
                _ck(L.moty_cuda_mat_apply_dev(l.v.h, p(self.vb), p(self.nrm), S, sh))
                qp, kp, vp = p(self.qb), p(self.kb), p(self.vb)
            if pos_dev is None:
                _ck(L.moty_cuda_attn_core_dev(a.h, p(self.ctx), qp, kp, vp, S, pos_base, sh))
            else:
                _ck(L.moty_cuda_attn_core_posdev(a.h, p(self.ctx), qp, kp, vp, S, p(pos_dev), pos_base, sh))
            _ck(L.moty_cuda_mat_apply_dev(l.o.h, p(self.tmp), p(self.ctx), S, sh))
            if fold_ffn[i]:
                _ck(L.moty_cuda_ffn_resnorm_dev(l.gate.h, l.up.h, l.down.h, ACT_SILU, p(self.tmp), p(x), p(self.tmp), None, p(x_alt),
                                                p(post_ln), eps, sh))
                x, x_alt = x_alt, x
            else:
                _ck(L.moty_cuda_add_rmsnorm_dev(p(x), p(self.tmp), p(self.nrm), p(post_ln), S, D, eps, sh))
                if l.moe is not None:
                    _ck(L.moty_cuda_moe_apply_dev(l.moe.h, p(self.tmp), p(self.nrm), S, None, 0, l.norm_topk, None, None, sh))
                else:
                    _ck(L.moty_cuda_ffn_dev(l.gate.h, l.up.h, l.down.h, ACT_SILU, p(self.tmp), p(self.nrm), S, sh))
            if i + 1 < nl and fold_qkv[i + 1]:
                pending = True
            elif i + 1 < nl:
                _ck(L.moty_cuda_add_rmsnorm_dev(p(x), p(self.tmp), p(self.nrm), p(self.ln[i + 1][0]), S, D, eps, sh))
            else:
                _ck(L.moty_cuda_add_dev(p(x), p(self.tmp), C.c_longlong(S * D), sh))
        return x

    def _decode_body(self, sh):
        """One greedy step with everything on the device: the token comes from ``self.ids[0]``, the position from
        ``self.pos_dev``; the new token goes to ``self.ids[0]`` and ``self.hist[self.cnt]``, position and count move on."""
        L, D = lib(), self.D
        p = lambda ten: C.c_void_p(ten.data_ptr())
        _ck(L.moty_cuda_embed_rows_dev(self.head.h, p(self.x), p(self.ids), 1, C.c_float(1.0), sh))
        x = self._layers(1, self.max_t - 1, self.pos_dev, sh)
        _ck(L.moty_cuda_rmsnorm_dev(p(self.nrm), p(x), p(self.final_norm), 1, D, C.c_float(self.eps), sh))
        _ck(L.moty_cuda_head_argmax_dev(self.head.h, p(self.nrm), 1, p(self.out_id), p(self.logits), sh))
        self.ids[:1].copy_(self.out_id)
        self.hist.index_copy_(0, self.cnt, self.out_id)
        self.pos_dev += 1
        self.cnt += 1

    def greedy_graph(self, first_tok, pos0, n):
        """n greedy tokens after ``first_tok`` at position pos0, the decode step captured ONCE into a CUDA graph and
        replayed n times (the attention core reads its position from the device).  Returns the n token ids."""
        t = self.torch
        if pos0 + n > self.max_t:
            raise MotyCudaError(f"positions {pos0}..{pos0 + n} exceed the cache of {self.max_t}")
        if getattr(self, "pos_dev", None) is None:                       # persistent: the captured graph holds their addresses
            self.pos_dev = t.zeros((1,), device=self.dev, dtype=t.int32)
            self.cnt = t.zeros((1,), device=self.dev, dtype=t.int64)
            self.hist = t.zeros((self.max_t + 1,), device=self.dev, dtype=t.int32)

        def reset(tok, pos):
            self.ids[:1].fill_(int(tok)); self.pos_dev.fill_(int(pos)); self.cnt.zero_()

        if getattr(self, "_graph", None) is None:
            with t.cuda.stream(self.stream):                             # one plain run first: scratch buffers, kernel attributes
                reset(first_tok, pos0)
                self._decode_body(C.c_void_p(stream_handle(self.stream)))
            self.stream.synchronize()
            # from here on the library's scratch may not move: the graph holds its addresses
            self._hold_scratch(1)
            try:
                g = t.cuda.CUDAGraph()
                with t.cuda.graph(g, stream=self.stream):
                    self._decode_body(C.c_void_p(stream_handle(t.cuda.current_stream())))
            except BaseException:
                self._hold_scratch(-1)
                raise
            self._graph = g
        with t.cuda.stream(self.stream):
            reset(first_tok, pos0)
            for _ in range(n):
                self._graph.replay()
        self.stream.synchronize()
        self._check_kernels()
        return [int(v) for v in self.hist[:n].cpu().numpy()]

    def close(self):
        self._drop_graph()                       # lifts the scratch freeze taken for the captured step
        for a in self.attn:
            a.close()

    def __del__(self):
        try:
            self._drop_graph()
        except Exception:
            pass


class GemmaLayer:
    """One layer of the reference's ``gemma`` engine (engines/gemma.c:299-386, :392-401, :466-483): int8 matrices
    (q, k, v, o, gate, up, down; optionally the rows of q, k and v in one matrix), the four sandwich norms and the three
    per-head norms as MULTIPLIERS (1 + w for a zero-centred checkpoint), and the layer's own attention geometry: a
    sliding layer has ``window`` > 0 and rotates every pair (``rot`` = head_dim / 2); a global one has ``window`` = 0,
    its own head_dim / KV-head count / theta, and ``rot`` rotated pairs of the p-RoPE."""

    def __init__(self, q, k, v, o, gate, up, down, in_ln, post_attn_ln, pre_ff_ln, post_ff_ln, qn, kn, vn=None, *, n_kv_heads, head_dim,
                 theta, window=0, rot=None, scale=0.0, qkv=None):
        self.q, self.k, self.v, self.o, self.gate, self.up, self.down, self.qkv = q, k, v, o, gate, up, down, qkv
        self.in_ln, self.post_attn_ln, self.pre_ff_ln, self.post_ff_ln = in_ln, post_attn_ln, pre_ff_ln, post_ff_ln
        self.qn, self.kn, self.vn = qn, kn, vn
        self.KV, self.hd, self.theta, self.window, self.scale = n_kv_heads, head_dim, float(theta), int(window), float(scale)
        self.rot = head_dim // 2 if rot is None else int(rot)


class GemmaDecoder(DenseDecoder):
    """The step of engines/gemma.c:453-497 without the per-layer-embedding branch (ple_dim = 0) and without shared KV
    layers: embedding rows scaled by sqrt(hidden), per layer  x += post_attn_norm(attn(in_norm(x)))  and
    x += post_ff_norm(gelu_mlp(pre_ff_norm(x))), the final norm of the last token, the lm_head and the greedy pick.
    The final logit soft-cap (softcap * tanhf(logit / softcap)) is monotonic, so the greedy pick is taken from the
    uncapped logits; ``step(..., want_logits=True)`` returns them uncapped."""

    def __init__(self, layers, head: Mat, final_norm, n_heads, max_t, eps=1e-6, kv8=False, device=0, max_S=64, fold_addnorm=False,
                 fold_ffn=False):
        # the folds of the sandwich steps into their consumers are built and bit-identical, and off by default: at hidden
        # 3840 they measured a loss (289 -> 263 tok/s replayed on the 48-layer shape; every CTA of the consumer redoes two
        # reductions over the row, where the separate one-CTA launch is nearly free under programmatic dependent launch)
        import torch
        self.torch = torch
        self.dev = torch.device(f"cuda:{device}")
        self.layers, self.head = layers, head
        self.H, self.eps, self.max_t = n_heads, float(eps), max_t
        self.D = head.I
        self.embed_scale = float(np.sqrt(np.float32(self.D)))
        self.fold_addnorm, self.fold_ffn = bool(fold_addnorm), bool(fold_ffn)
        f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(self.dev)
        self.final_norm = f(final_norm)
        self.ln = [tuple(f(g) for g in (l.in_ln, l.post_attn_ln, l.pre_ff_ln, l.post_ff_ln)) for l in layers]
        self.attn = [Attn(n_heads, l.KV, l.hd, max_t, theta=l.theta, eps=eps, rot=l.rot, qn=l.qn, kn=l.kn, vn=l.vn, kv8=kv8,
                          device=device, gemma=True, window=l.window, scale=l.scale) for l in layers]
        # buffers sized for the widest layer
        self.hd, self.KV = max(l.hd for l in layers), 0
        self._qw = max(n_heads * l.hd for l in layers)
        self._kw = max(l.KV * l.hd for l in layers)
        self.stream = torch.cuda.Stream(device=self.dev)
        self._alloc(max_S)

    def _alloc(self, S):
        t, dev = self.torch, self.dev
        e = lambda *shape: t.empty(shape, device=dev, dtype=t.float32)
        self._drop_graph()
        self.cap = 0                             # until all of them are there: a failed allocation must not leave small ones for S rows
        self.x, self.nrm, self.tmp = e(S, self.D), e(S, self.D), e(S, self.D)
        self.x_alt = e(1, self.D)
        self.qb, self.kb, self.vb, self.ctx = e(S, self._qw), e(S, self._kw), e(S, self._kw), e(S, self._qw)
        self.qkvb = e(1, self._qw + 2 * self._kw)
        self.ids = t.empty((S,), device=dev, dtype=t.int32)
        self.out_id = t.empty((1,), device=dev, dtype=t.int32)
        self.logits = e(1, self.head.O)
        self.cap = S

    def _embed(self, S, sh):
        p = lambda ten: C.c_void_p(ten.data_ptr())
        _ck(lib().moty_cuda_embed_rows_dev(self.head.h, p(self.x), p(self.ids), S, C.c_float(self.embed_scale), sh))

    def _layers(self, S, pos_base, pos_dev, sh):
        """engines/gemma.c:466-483 on self.x [S][D]; on return self.nrm holds the FINAL norm of every row (the last
        sandwich step opens it), so the caller goes straight to the lm_head.  With one token the sandwich steps in front
        of the fused [q|k|v] product and in front of the FFN block ride inside those launches (same bits)."""
        L, D, eps = lib(), self.D, C.c_float(self.eps)
        p = lambda ten: C.c_void_p(ten.data_ptr())
        nl = len(self.layers)
        x, x_alt = self.x, self.x_alt
        one = self.fold_addnorm and S == 1
        fold_qkv = [one and l.qkv is not None and bool(L.moty_cuda_mat_addnorm_supported(l.qkv.h)) for l in self.layers]
        fold_ffn = [self.fold_ffn and S == 1 and bool(L.moty_cuda_ffn_resnorm_supported(l.gate.h, l.up.h)) for l in self.layers]
        pending = None                           # gains of the post-FFN norm whose sandwich step is still owed (t in self.tmp)
        _ck(L.moty_cuda_rmsnorm_dev(p(self.nrm), p(x), p(self.ln[0][0]), S, D, eps, sh))
        for i, (l, (in_ln, post_attn, pre_ff, post_ff), a) in enumerate(zip(self.layers, self.ln, self.attn)):
            qw, kw = self.H * l.hd, l.KV * l.hd
            if S == 1 and l.qkv is not None:
                if pending is not None:
                    _ck(L.moty_cuda_mat_apply_resnorm_dev(l.qkv.h, p(self.qkvb), p(x), p(self.tmp), p(pending), p(x_alt), p(in_ln), eps, sh))
                    x, x_alt = x_alt, x
                    pending = None
                else:
                    _ck(L.moty_cuda_mat_apply_dev(l.qkv.h, p(self.qkvb), p(self.nrm), 1, sh))
                base = self.qkvb.data_ptr()
                qp, kp, vp = C.c_void_p(base), C.c_void_p(base + 4 * qw), C.c_void_p(base + 4 * (qw + kw))
            else:
                _ck(L.moty_cuda_mat_apply_dev(l.q.h, p(self.qb), p(self.nrm), S, sh))
                _ck(L.moty_cuda_mat_apply_dev(l.k.h, p(self.kb), p(self.nrm), S, sh))
                _ck(L.moty_cuda_mat_apply_dev(l.v.h, p(self.vb), p(self.nrm), S, sh))
                qp, kp, vp = p(self.qb), p(self.kb), p(self.vb)
            if pos_dev is None:
                _ck(L.moty_cuda_attn_core_dev(a.h, p(self.ctx), qp, kp, vp, S, pos_base, sh))
            else:
                _ck(L.moty_cuda_attn_core_posdev(a.h, p(self.ctx), qp, kp, vp, S, p(pos_dev), pos_base, sh))
            _ck(L.moty_cuda_mat_apply_dev(l.o.h, p(self.tmp), p(self.ctx), S, sh))
            if fold_ffn[i]:
                _ck(L.moty_cuda_ffn_resnorm_dev(l.gate.h, l.up.h, l.down.h, ACT_GELU_TANH, p(self.tmp), p(x), p(self.tmp), p(post_attn),
                                                p(x_alt), p(pre_ff), eps, sh))
                x, x_alt = x_alt, x
            else:
                _ck(L.moty_cuda_normadd_rmsnorm_dev(p(x), p(self.tmp), p(post_attn), p(self.nrm), p(pre_ff), S, D, eps, sh))
                _ck(L.moty_cuda_ffn_dev(l.gate.h, l.up.h, l.down.h, ACT_GELU_TANH, p(self.tmp), p(self.nrm), S, sh))
            if i + 1 < nl and fold_qkv[i + 1]:
                pending = post_ff
            else:
                nxt = self.ln[i + 1][0] if i + 1 < nl else self.final_norm
                _ck(L.moty_cuda_normadd_rmsnorm_dev(p(x), p(self.tmp), p(post_ff), p(self.nrm), p(nxt), S, D, eps, sh))
        return x

    def step(self, ids, pos_base, want_logits=False):
        t, L = self.torch, lib()
        ids = np.ascontiguousarray(ids, np.int32).ravel()
        S = ids.size
        if S > getattr(self, "_max_S", 0):
            self._drop_graph()
            self._max_S = S
        if S > self.cap:
            self._alloc(S)
        if pos_base + S > self.max_t:
            raise MotyCudaError(f"positions {pos_base}..{pos_base + S} exceed the cache of {self.max_t}")
        p = lambda ten: C.c_void_p(ten.data_ptr())
        with t.cuda.stream(self.stream):
            sh = C.c_void_p(stream_handle(self.stream))
            self.ids[:S].copy_(t.from_numpy(ids), non_blocking=True)
            self._embed(S, sh)
            self._layers(S, pos_base, None, sh)
            _ck(L.moty_cuda_head_argmax_dev(self.head.h, p(self.nrm[S - 1:S]), 1, p(self.out_id), p(self.logits), sh))
            tok = int(self.out_id.cpu()[0])
            self._check_kernels()
            if want_logits:
                return tok, self.logits.cpu().numpy()[0]
        return tok

    def prefill(self, ids, pos_base=0, block=512):
        """A long prompt in blocks of ``block`` tokens (the blocked prefill of engines/gemma.c:484-485: the blocks
        before the last need no logits); returns the greedy token after the last one."""
        ids = np.ascontiguousarray(ids, np.int32).ravel()
        tok = None
        for lo in range(0, ids.size, block):
            tok = self.step(ids[lo:lo + block], pos_base + lo)
        return tok

    def _decode_body(self, sh):
        L = lib()
        p = lambda ten: C.c_void_p(ten.data_ptr())
        self._embed(1, sh)
        self._layers(1, self.max_t - 1, self.pos_dev, sh)
        _ck(L.moty_cuda_head_argmax_dev(self.head.h, p(self.nrm), 1, p(self.out_id), p(self.logits), sh))
        self.ids[:1].copy_(self.out_id)
        self.hist.index_copy_(0, self.cnt, self.out_id)
        self.pos_dev += 1
        self.cnt += 1


class PagedDecoder(DenseDecoder):
    """Several sequences of one dense (or routed) model at once over a paged 4-bit KV cache (``moty_b200.Kv4``): prompts
    and single tokens of any mix of sequences go through the layers as one batch of rows; sequences can be forked (full
    pages shared, the last one copied), ended, and the pages in use moved together.  The layer order is DenseDecoder's;
    only the attention core differs (append_rope + attend on the pages instead of ``Attn``).

    ``pages``: pages of 64 positions in the pool (all layers of a position lie in one page).  ``max_pages``: the most a
    sequence may hold.  A call that raises (the pool is out of pages, an allocation or a launch fails, a kernel reports an
    error) leaves lengths, pages and books as they were (``compact`` says what happens there)."""

    def __init__(self, layers, head: Mat, final_norm, n_heads, n_kv_heads, head_dim, pages, max_seqs=64, max_pages=64, theta=1e6, eps=1e-6,
                 rot=None, device=0, max_S=64):
        import torch
        self.torch = torch
        self.dev = torch.device(f"cuda:{device}")
        self.layers, self.head = layers, head
        self.H, self.KV, self.hd, self.eps = n_heads, n_kv_heads, head_dim, float(eps)
        self.theta, self.rot = float(theta), head_dim if rot is None else rot
        self.D = head.I
        f = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(self.dev)
        self.final_norm = f(final_norm)
        self.ln = [(f(l.in_ln), f(l.post_ln)) for l in layers]
        self.qk_gain = [(f(l.qn), f(l.kn)) for l in layers]
        self.kv = Kv4(len(layers), n_kv_heads, head_dim, pages, device=device)
        self.max_seqs, self.max_pages = max_seqs, max_pages
        self.table = np.full((max_seqs, max_pages), -1, np.int32)        # row = sequence id
        self.lens = np.zeros(max_seqs, np.int32)
        self.used = np.zeros(max_seqs, bool)
        self._broken = False
        self.stream = torch.cuda.Stream(device=self.dev)
        self._alloc(max_S)

    def _alloc(self, S):
        t, dev = self.torch, self.dev
        qw, kw = self.H * self.hd, self.KV * self.hd
        e = lambda *shape: t.empty(shape, device=dev, dtype=t.float32)
        self._drop_graph()
        self.cap = 0                             # until all of them are there: a failed allocation must not leave small ones for S rows
        self.x, self.nrm, self.tmp, self.ctx = e(S, self.D), e(S, self.D), e(S, self.D), e(S, qw)
        self.qkvb = e(S, qw + 2 * kw)
        self.ids = t.empty((S,), device=dev, dtype=t.int32)
        self.out_id = t.empty((S,), device=dev, dtype=t.int32)
        self.logits = None
        self.cap = S

    # -- sequences ------------------------------------------------------------------------------------------------------
    def new(self) -> int:
        """An empty sequence; returns its id."""
        self._usable()
        free = np.flatnonzero(~self.used)
        if not free.size:
            raise MotyCudaError(f"all {self.max_seqs} sequences are in use")
        self.used[free[0]] = True
        return int(free[0])

    def end(self, sid) -> None:
        """Forget a sequence; pages it does not share are free again."""
        self._check(sid)
        self._drop_graph()
        self.kv.release(self.table[sid])
        self.table[sid] = -1; self.lens[sid] = 0; self.used[sid] = False

    def fork(self, sid, n=1) -> list:
        """n copies of a sequence: they share its full pages, the last partial page is copied on the device."""
        self._check(sid)
        if n < 1:
            raise MotyCudaError(f"{n} forks")
        self._drop_graph()
        L = int(self.lens[sid]); full = L // Kv4.PAGE
        free = np.flatnonzero(~self.used)[:n]
        if free.size < n:
            raise MotyCudaError(f"{n} forks, {free.size} sequences free")
        fresh = self.kv.alloc(n) if L % Kv4.PAGE else np.full(n, -1, np.int32)
        t = self.torch
        try:
            with t.cuda.stream(self.stream):
                up = lambda a: t.from_numpy(np.ascontiguousarray(a, np.int32)).to(self.dev)
                table, lens = up(self.table), up(self.lens)
                src, dst, new = up(np.full(n, sid)), up(free), up(fresh)
                self.kv.fork_dev(n, src.data_ptr(), dst.data_ptr(), new.data_ptr(), self.max_seqs, lens.data_ptr(), table.data_ptr(),
                                 self.max_pages, stream=stream_handle(self.stream))
                table, lens = table.cpu().numpy(), lens.cpu().numpy()
                self._check_kernels()
            self.kv.retain(np.tile(self.table[sid, :full], n))       # all or none
        except BaseException:
            self._settle()
            self.kv.release(fresh)
            raise
        self.table, self.lens = table, lens
        self.used[free] = True
        return [int(s) for s in free]

    def compact(self) -> int:
        """Move the pages in use to the lowest ids; returns how many moved.  Should the moves themselves fail, the books already
        name the new places: the decoder refuses every further call then."""
        self._usable()
        self._drop_graph()
        t = self.torch
        with t.cuda.stream(self.stream):         # what can fail for want of memory comes before the books change
            table = t.from_numpy(self.table).to(self.dev)
            moves = t.empty((2, self.kv.pages), device=self.dev, dtype=t.int32)
            src, dst = self.kv.compact_plan()
            n = int(src.size)
            if not n:
                return 0
            try:
                moves[0, :n].copy_(t.from_numpy(src)); moves[1, :n].copy_(t.from_numpy(dst))
                self.kv.compact_dev(n, moves[0].data_ptr(), moves[1].data_ptr(), table.numel(), table.data_ptr(), table.data_ptr(),
                                    stream=stream_handle(self.stream))
                table = table.cpu().numpy()
                self._check_kernels()
            except BaseException:
                self._broken = True
                raise
        self.table = table
        return n

    def _usable(self):
        if self._broken:
            raise MotyCudaError("a compaction failed: the pages no longer fit the sequences")

    def _check(self, sid):
        self._usable()
        if not (0 <= sid < self.max_seqs and self.used[sid]):
            raise MotyCudaError(f"sequence {sid} is not in use")

    def _check_tokens(self, toks):
        for i in toks:
            if i.min() < 0 or i.max() >= self.head.O:
                raise MotyCudaError(f"a token id outside the vocabulary of {self.head.O}")

    @contextlib.contextmanager
    def _taken(self, sids, more):
        """Pages for `more[i]` further positions of each sequence: all of them or none, and none again where the block fails."""
        grow = []
        for s, n in zip(sids, more):
            have, want = -(-int(self.lens[s]) // Kv4.PAGE), -(-(int(self.lens[s]) + int(n)) // Kv4.PAGE)
            if want > self.max_pages:
                raise MotyCudaError(f"sequence {s} would hold {want} pages, more than {self.max_pages}")
            grow.append([p for p in range(have, want) if self.table[s, p] < 0])
        ids = self.kv.alloc(sum(map(len, grow)))
        at = 0
        for s, g in zip(sids, grow):
            self.table[s, g] = ids[at:at + len(g)]; at += len(g)
        try:
            yield
        except BaseException:
            self._settle()
            for s, g in zip(sids, grow):
                self.table[s, g] = -1
            self.kv.release(ids)
            raise

    def _settle(self):
        """After a failure: what is still on its way is done with the pages before others get them."""
        try:
            self.stream.synchronize()
        except Exception:
            pass

    # -- steps ----------------------------------------------------------------------------------------------------------
    def run(self, batch, want_logits=False):
        """batch: [(sequence id, token ids), ...], each sequence once.  Appends every sequence's tokens to it and returns the
        greedy next token after the last of each (and those rows' logits when asked)."""
        t, L = self.torch, lib()
        sids = [int(s) for s, _ in batch]
        toks = [np.ascontiguousarray(i, np.int32).ravel() for _, i in batch]
        for s in sids:
            self._check(s)
        if len(set(sids)) != len(sids) or any(not i.size for i in toks):
            raise MotyCudaError("each sequence of a batch once, with at least one token")
        self._check_tokens(toks)
        counts = [i.size for i in toks]
        S, n = sum(counts), len(sids)
        with self._taken(sids, counts):
            self._drop_graph()                   # a batch of another shape may grow the library's scratch
            if S > self.cap:
                self._alloc(S)
            lens = self.lens[sids] + np.array(counts, np.int32)
            row0 = np.concatenate([[0], np.cumsum(counts)])
            with t.cuda.stream(self.stream):
                up = lambda a: t.from_numpy(np.ascontiguousarray(a, np.int32)).to(self.dev)
                d_row0, d_len, d_tab = up(row0), up(lens), up(self.table[sids])
                b = Kv4Batch(n, S, d_row0.data_ptr(), d_len.data_ptr(), d_tab.data_ptr(), self.max_pages, max_rows=max(counts),
                             max_len=int(lens.max()))
                self.ids[:S].copy_(t.from_numpy(np.concatenate(toks)))
                self._embed_rows(S)
                self._layers_paged(S, b)
                last = self.x[:S].index_select(0, (d_row0[1:] - 1).long())
                logits = t.empty((n, self.head.O), device=self.dev, dtype=t.float32)
                self._head(last, n, logits)
                out = self.out_id[:n].cpu().numpy().copy()
                self._check_kernels()
                if want_logits:
                    logits = logits.cpu().numpy()
            self.lens[sids] = lens               # nothing can fail from here on
        return (out, logits) if want_logits else out

    def greedy(self, sids, tokens, n):
        """n greedy tokens for each of the sequences after ``tokens``, the step captured ONCE into a CUDA graph and replayed
        (lengths move on the device).  Returns int32 [len(sids)][n]."""
        t = self.torch
        sids = [int(s) for s in sids]
        for s in sids:
            self._check(s)
        if len(set(sids)) != len(sids) or not sids or n < 1:
            raise MotyCudaError("each sequence once, at least one, and at least one token")
        k = len(sids)
        tokens = np.ascontiguousarray(tokens, np.int32).ravel()
        if tokens.size != k:
            raise MotyCudaError(f"{tokens.size} tokens for {k} sequences")
        self._check_tokens([tokens])
        with self._taken(sids, [n] * k):
            if k > self.cap:
                self._alloc(k)
            self._drop_graph()
            start = self.lens[sids].copy()
            with t.cuda.stream(self.stream):
                up = lambda a: t.from_numpy(np.ascontiguousarray(a, np.int32)).to(self.dev)
                row0, tab, lens = up(np.arange(k + 1)), up(self.table[sids]), up(start)
                first = up(tokens)
                hist, cnt = t.zeros((n + 1, k), device=self.dev, dtype=t.int32), t.zeros((1,), device=self.dev, dtype=t.int64)
                logits = t.empty((k, self.head.O), device=self.dev, dtype=t.float32)
                b = Kv4Batch(k, k, row0.data_ptr(), lens.data_ptr(), tab.data_ptr(), self.max_pages, max_rows=1, max_len=int(start.max()) + n)

                def body():
                    lens.add_(1)
                    self._embed_rows(k)
                    self._layers_paged(k, b)
                    self._head(self.x[:k], k, logits)
                    self.ids[:k].copy_(self.out_id[:k])
                    hist.index_copy_(0, cnt, self.out_id[:k].view(1, k))
                    cnt.add_(1)

                def reset():
                    self.ids[:k].copy_(first); lens.copy_(up(start)); cnt.zero_()

                reset()
                body()                               # one plain run: scratch, kernel attributes (its rows are written again below)
            # (the scratch is neither frozen nor set free here: this graph does not outlive the call, and another decoder's captured
            # step may be relying on the freeze that it took)
            self.stream.synchronize()
            g = t.cuda.CUDAGraph()
            with t.cuda.graph(g, stream=self.stream):
                body()
            with t.cuda.stream(self.stream):
                reset()
                for _ in range(n):
                    g.replay()
            self.stream.synchronize()
            self._check_kernels()
            del g
            out = hist[:n].cpu().numpy().T.copy()
            self.lens[sids] += n                     # nothing can fail from here on
        return out

    def _embed_rows(self, S):
        p = lambda ten: C.c_void_p(ten.data_ptr())
        _ck(lib().moty_cuda_embed_rows_dev(self.head.h, p(self.x), p(self.ids), S, C.c_float(1.0), C.c_void_p(stream_handle(self.torch.cuda.current_stream()))))

    def _head(self, rows, n, logits):
        p = lambda ten: C.c_void_p(ten.data_ptr())
        sh = C.c_void_p(stream_handle(self.torch.cuda.current_stream()))
        _ck(lib().moty_cuda_rmsnorm_dev(p(self.nrm), p(rows), p(self.final_norm), n, self.D, C.c_float(self.eps), sh))
        _ck(lib().moty_cuda_head_argmax_dev(self.head.h, p(self.nrm), n, p(self.out_id), p(logits), sh))

    def _layers_paged(self, S, b):
        """DenseDecoder._layers on self.x [S][D] with the rows' attention on the pages."""
        L, D, eps = lib(), self.D, C.c_float(self.eps)
        stream = stream_handle(self.torch.cuda.current_stream())
        sh = C.c_void_p(stream)
        p = lambda ten: C.c_void_p(ten.data_ptr())
        qw, kw = self.H * self.hd, self.KV * self.hd
        nl = len(self.layers)
        _ck(L.moty_cuda_rmsnorm_dev(p(self.nrm), p(self.x), p(self.ln[0][0]), S, D, eps, sh))
        base = self.qkvb.data_ptr()
        for i, (l, (in_ln, post_ln), (qn, kn)) in enumerate(zip(self.layers, self.ln, self.qk_gain)):
            if l.qkv is not None:                # one product, rows [q | k | v]
                _ck(L.moty_cuda_mat_apply_dev(l.qkv.h, p(self.qkvb), p(self.nrm), S, sh))
                qp, kp, vp, ldq, ldk = base, base + 4 * qw, base + 4 * (qw + kw), qw + 2 * kw, qw + 2 * kw
            else:
                qp, kp, vp, ldq, ldk = base, base + 4 * S * qw, base + 4 * S * (qw + kw), 0, 0
                for m, ptr in ((l.q, qp), (l.k, kp), (l.v, vp)):
                    _ck(L.moty_cuda_mat_apply_dev(m.h, C.c_void_p(ptr), p(self.nrm), S, sh))
            self.kv.append_rope_dev(i, self.H, qp, kp, vp, b, self.rot, self.theta, self.eps, qn.data_ptr() if qn is not None else 0,
                                    kn.data_ptr() if kn is not None else 0, stream=stream, q_ld=ldq, kv_ld=ldk)
            self.kv.attend_dev(i, self.ctx.data_ptr(), qp, self.H, b, stream=stream, q_ld=ldq)
            _ck(L.moty_cuda_mat_apply_dev(l.o.h, p(self.tmp), p(self.ctx), S, sh))
            _ck(L.moty_cuda_add_rmsnorm_dev(p(self.x), p(self.tmp), p(self.nrm), p(post_ln), S, D, eps, sh))
            if l.moe is not None:
                _ck(L.moty_cuda_moe_apply_dev(l.moe.h, p(self.tmp), p(self.nrm), S, None, 0, l.norm_topk, None, None, sh))
            else:
                _ck(L.moty_cuda_ffn_dev(l.gate.h, l.up.h, l.down.h, ACT_SILU, p(self.tmp), p(self.nrm), S, sh))
            if i + 1 < nl:
                _ck(L.moty_cuda_add_rmsnorm_dev(p(self.x), p(self.tmp), p(self.nrm), p(self.ln[i + 1][0]), S, D, eps, sh))
            else:
                _ck(L.moty_cuda_add_dev(p(self.x), p(self.tmp), C.c_longlong(S * D), sh))

    def close(self):
        self._drop_graph()
        self.kv.close()
