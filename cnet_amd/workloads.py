"""Multi-layer workloads of the benchmark configurations, expressed as sequences of C-ABI calls (orchestration only).

TokenModel is the complex token model of the fifth configuration: embedding -> DFT along the sequence axis -> Hadamard gate
with shared complex weights -> Linear, CGelu, Linear -> Linear to vocabulary logits -> CrossEntropy on the next token.
Upstream has no transform along an inner axis; its oracle is FourierTrans(seq) applied to every (sequence, channel) column.
Next-token labels: position t of a sequence is labelled with token t+1; the last position wraps to the first token.
"""
import ctypes as C

import numpy as np

from . import capi, ops


class TokenModel:
    def __init__(self, batch, seq, dim, hidden, vocab, params, conjugate_pairs=False):
        """params: dict of host arrays: table (2,V,D), gate (2,D), w1 (2,H,D), w2 (2,D,H), w3 (2,V,D).
        conjugate_pairs: the loss is real, so every dz* gradient is the conjugate of the dz gradient; the Linear backward
        passes then compute the dz products only and write the dz* halves as their conjugates, and of the sequence-axis
        transform only the dz* product is formed (its one consumer, the embedding table, gathers dz* alone)."""
        self.conjugate_pairs = conjugate_pairs
        self.B, self.S, self.D, self.H, self.V = batch, seq, dim, hidden, vocab
        self.rows = batch * seq
        p = {k: ops.CMat.from_host(v[0], v[1]) for k, v in params.items()}
        self.table, self.gate, self.w1, self.w2, self.w3 = p["table"], p["gate"], p["w1"], p["w2"], p["w3"]
        capi.call("cnet_cdft_plan", seq)
        fr, fi = C.c_void_p(), C.c_void_p()
        capi.call("cnet_cdft_twiddle", seq, C.byref(fr), C.byref(fi))
        ld = (seq + 3) // 4 * 4
        self.F = ops.CMat(ops.Plane(fr.value, seq, seq, ld), ops.Plane(fi.value, seq, seq, ld))
        R, D, H, V = self.rows, dim, hidden, vocab
        E = ops.CMat.empty
        G = ops.Grad.empty
        self.x, self.m, self.h = E(R, D), E(R, D), E(R, D)
        self.u, self.a, self.o, self.logits = E(R, H), E(R, H), E(R, D), E(R, V)
        self.s, self.loss, self.argmax = capi.empty(R), capi.empty(R), capi.empty(R, np.int32)
        self.d_logits, self.d_o, self.d_a, self.d_u = G(R, V), G(R, D), G(R, H), G(R, H)
        self.d_h, self.d_m, self.d_x = G(R, D), G(R, D), G(R, D)
        self.d_w1, self.d_w2, self.d_w3, self.d_gate = G(H, D), G(D, H), G(V, D), G(1, D)
        self.d_table_re, self.d_table_im = ops.Plane.empty(V, D), ops.Plane.empty(V, D)
        self.tokens = self.labels = None

    def set_tokens(self, ids):
        ids = np.ascontiguousarray(ids, np.int32).reshape(self.B, self.S)
        self.tokens = ops.ints(ids)
        self.labels = ops.ints(np.roll(ids, -1, axis=1).reshape(-1))
        return self

    def forward(self):
        B, S, D = self.B, self.S, self.D
        xb = ops.CMat(ops.Plane(self.x.re.ptr, B, S * D, S * D), ops.Plane(self.x.im.ptr, B, S * D, S * D))
        ops.embedding_fwd(self.table, self.tokens, xb, S)
        # M_b = F X_b for every sequence b: one strided-batched launch, F shared (stride 0)
        ops.cgemm_batched(self.F, 0, self.x, S * D, self.m, S * D, S, D, S, B, a_kmajor=0, b_kmajor=1)
        ops.hadamard_fwd(self.m, self.gate, self.h, shared=True)
        ops.linear_gelu_fwd(self.h, self.w1, self.u, self.a)   # the CGelu applied where the product is stored
        ops.linear_fwd(self.a, self.w2, self.o)
        ops.linear_fwd(self.o, self.w3, self.logits)
        ops.cross_entropy_fwd(self.logits, self.labels, self.s, self.loss, self.argmax, None)

    def backward(self):
        B, S, D = self.B, self.S, self.D
        if self.conjugate_pairs:
            # one gradient per value: every pass reads the dz planes only; the dz* planes are written where something reads
            # them (parameter gradients, and d_m, whose dz* half feeds the sequence transform)
            ops.cross_entropy_bwd_sym(self.logits, self.s, self.labels, self.d_logits, mirror=False)
            ops.linear_bwd_input_sym(self.d_logits, self.w3, self.d_o, mirror=False)
            ops.linear_bwd_weight_sym(self.d_logits, self.o, self.d_w3)
            ops.linear_bwd_input_sym(self.d_o, self.w2, self.d_a, mirror=False)
            ops.linear_bwd_weight_sym(self.d_o, self.a, self.d_w2)
            ops.gelu_bwd_sym(self.u, self.d_a, self.d_u, mirror=False)
            ops.linear_bwd_input_sym(self.d_u, self.w1, self.d_h, mirror=False)
            ops.linear_bwd_weight_sym(self.d_u, self.h, self.d_w1)
            ops.hadamard_bwd_sym(self.m, self.gate, self.d_h, self.d_m, self.d_gate, shared=True)
        else:
            ops.cross_entropy_bwd(self.logits, self.s, self.labels, self.d_logits)
            ops.linear_bwd_input(self.d_logits, self.w3, self.d_o)
            ops.linear_bwd_weight(self.d_logits, self.o, self.d_w3)
            ops.linear_bwd_input(self.d_o, self.w2, self.d_a)
            ops.linear_bwd_weight(self.d_o, self.a, self.d_w2)
            ops.gelu_bwd(self.u, self.d_a, self.d_u)
            ops.linear_bwd_input(self.d_u, self.w1, self.d_h)
            ops.linear_bwd_weight(self.d_u, self.h, self.d_w1)
            ops.hadamard_bwd(self.m, self.gate, self.d_h, self.d_m, self.d_gate, shared=True)
        # dz_b = F dM_b.dz ; dz*_b = conj(F) dM_b.dz*   (F symmetric)
        gdz = ops.CMat(self.d_m.planes[0], self.d_m.planes[1])
        gds = ops.CMat(self.d_m.planes[2], self.d_m.planes[3])
        xdz = ops.CMat(self.d_x.planes[0], self.d_x.planes[1])
        xds = ops.CMat(self.d_x.planes[2], self.d_x.planes[3])
        if not self.conjugate_pairs:
            ops.cgemm_batched(self.F, 0, gdz, S * D, xdz, S * D, S, D, S, B, b_kmajor=1)
        ops.cgemm_batched(self.F, 0, gds, S * D, xds, S * D, S, D, S, B, b_kmajor=1, conj_a=1)
        gs_re = ops.Plane(self.d_x.planes[2].ptr, B, S * D, S * D)
        gs_im = ops.Plane(self.d_x.planes[3].ptr, B, S * D, S * D)
        ops.embedding_bwd(self.tokens, gs_re, gs_im, self.d_table_re, self.d_table_im, D, self.V, B, S)

    def gemm_flops(self):
        R, S, D, H, V, B = self.rows, self.S, self.D, self.H, self.V, self.B
        lin = 8.0 * R * (D * H + H * D + D * V)
        dft = 8.0 * B * S * S * D
        return 3 * lin + 2 * dft if self.conjugate_pairs else 5 * lin + 3 * dft  # the products that are executed


class BlockTokenModel:
    """A deep complex token model: embedding, then `layers` blocks on a residual path, a norm before and after each, and the
    vocabulary on top.

        h_0 = embedding, y_0 = w_0 .* h_0 / rms(h_0)
        f_l = W2_l gelu(W1_l (gate_l .* F y_l))                       F: the DFT along the sequence
        h_{l+1} = h_l + scale v_l .* f_l / rms(f_l),   y_{l+1} = w_{l+1} .* h_{l+1} / rms(h_{l+1})
        loss: CrossEntropy of y_L head^T against the next token (without the logits), or against a teacher's top entries

    step() runs forward and backward; gradients are conjugate pairs, parameters receive both halves (the table dz* alone, as the
    SGD step reads it)."""

    def __init__(self, batch, seq, dim, hidden, vocab, layers, params, scale=0.5, eps=1e-6):
        """params: dict of host arrays (2, ...): table (V, D), head (V, D), and lists norm (L + 1 of (1, D)), gate, after (L of (1, D)),
        w1 (L of (H, D)), w2 (L of (D, H))."""
        assert layers >= 1
        self.B, self.S, self.D, self.H, self.V, self.L = batch, seq, dim, hidden, vocab, layers
        self.scale, self.eps = scale, eps
        self.rows = R = batch * seq

        def mat(v):
            return ops.CMat.from_host(v[0], v[1])
        self.p = {k: [mat(x) for x in v] if isinstance(v, list) else mat(v) for k, v in params.items()}
        capi.call("cnet_cdft_plan", seq)
        fr, fi = C.c_void_p(), C.c_void_p()
        capi.call("cnet_cdft_twiddle", seq, C.byref(fr), C.byref(fi))
        ld = (seq + 3) // 4 * 4
        self.F = ops.CMat(ops.Plane(fr.value, seq, seq, ld), ops.Plane(fi.value, seq, seq, ld))
        E, G = ops.CMat.empty, ops.Grad.empty
        self.h = [E(R, dim) for _ in range(layers + 1)]
        self.y = [E(R, dim) for _ in range(layers + 1)]
        self.s2 = [capi.empty(R) for _ in range(layers + 1)]     # of the norms in front of the blocks and of the head
        self.s1 = [capi.empty(R) for _ in range(layers)]         # of the norms behind the blocks
        self.m, self.g, self.f = ([E(R, dim) for _ in range(layers)] for _ in range(3))
        self.u, self.a = ([E(R, hidden) for _ in range(layers)] for _ in range(2))
        self.s, self.loss, self.argmax = capi.empty(R), capi.empty(R), capi.empty(R, np.int32)
        # gradients: the dz planes of activations, both halves of parameters (and of the sequence transform's result)
        self.dy, self.df, self.dg = G(R, dim), G(R, dim), G(R, dim)
        self.dh = [G(R, dim), G(R, dim)]
        self.da, self.du = G(R, hidden), G(R, hidden)
        self.grads = {k: [G(x.rows, x.cols) for x in v] if isinstance(v, list) else G(v.rows, v.cols) for k, v in self.p.items()}
        self.logits = self.dlogits = None
        self.teacher = None

    def set_tokens(self, ids, labels=None):
        """labels: by default the next token, none for the last position; a negative label leaves a position out"""
        ids = np.ascontiguousarray(ids, np.int32).reshape(self.B, self.S)
        if labels is None:
            labels = np.concatenate([ids[:, 1:], np.full((self.B, 1), -1, np.int32)], axis=1)
        self.tokens = ops.ints(ids)
        self.labels = ops.ints(np.asarray(labels).reshape(-1))
        return self

    def set_teacher(self, ids, probs):
        """[rows][top] entries to learn from instead of the labels; None: the labels again"""
        if ids is None:
            self.teacher = None
            return self
        ids = np.ascontiguousarray(ids, np.int32).reshape(self.rows, -1)
        self.teacher = (ops.ints(ids), capi.to_device(np.ascontiguousarray(probs, np.float32).reshape(ids.shape)), ids.shape[1])
        if self.logits is None:
            self.logits, self.dlogits = ops.CMat.empty(self.rows, self.V), ops.Grad.empty(self.rows, self.V)
        return self

    def _blocks_forward(self):
        B, S, D, p = self.B, self.S, self.D, self.p
        h0 = self.h[0]
        ops.embedding_fwd(p["table"], self.tokens, ops.CMat(ops.Plane(h0.re.ptr, B, S * D, S * D), ops.Plane(h0.im.ptr, B, S * D, S * D)), S)
        ops.norm_gate_fwd(h0, p["norm"][0], self.y[0], self.s2[0], self.eps)
        for k in range(self.L):
            ops.cgemm_batched(self.F, 0, self.y[k], S * D, self.m[k], S * D, S, D, S, B, b_kmajor=1)
            ops.hadamard_fwd(self.m[k], p["gate"][k], self.g[k], shared=True)
            ops.linear_gelu_fwd(self.g[k], p["w1"][k], self.u[k], self.a[k])
            ops.linear_fwd(self.a[k], p["w2"][k], self.f[k])
            ops.norm_join_fwd(self.h[k], self.f[k], p["after"][k], self.scale, self.h[k + 1], self.s1[k], p["norm"][k + 1], self.y[k + 1],
                              self.s2[k + 1], self.eps)

    def score(self):
        """The most likely token of every position (argmax) with -log of its probability (loss)."""
        self._blocks_forward()
        ops.vocab_head_fwd(self.y[self.L], self.p["head"], None, self.s, self.loss, self.argmax)

    def step(self):
        """loss and every gradient of one batch"""
        B, S, D, L, p, d = self.B, self.S, self.D, self.L, self.p, self.grads
        self._blocks_forward()
        top = self.y[L]
        if self.teacher is not None:
            ids, probs, n = self.teacher
            ops.linear_fwd(top, p["head"], self.logits)
            ops.distill_fwd_bwd_sym(self.logits, ids, probs, n, self.s, self.loss, self.dlogits, mirror=False)
            ops.linear_bwd_sym(self.dlogits, top, p["head"], self.dy, d["head"], mirror_dx=False)
        else:
            ops.vocab_head_fwd_bwd_sym(top, p["head"], self.labels, self.s, self.loss, None, self.dy, d["head"], mirror_dx=False)
        dh = None
        for k in reversed(range(L)):
            below = self.dh[k % 2]
            # (the bottom one is written with both halves: the embedding gathers the dz* half)
            ops.norm_join_bwd_sym(self.f[k], self.s1[k], p["after"][k], self.scale, self.h[k + 1], self.s2[k + 1], p["norm"][k + 1], dh, self.dy,
                                  below, self.df, d["after"][k], d["norm"][k + 1], mirror=k == 0)
            ops.linear_bwd_input_sym(self.df, p["w2"][k], self.da, mirror=False)
            ops.linear_bwd_weight_sym(self.df, self.a[k], d["w2"][k])
            ops.gelu_bwd_sym(self.u[k], self.da, self.du, mirror=False)
            ops.linear_bwd_input_sym(self.du, p["w1"][k], self.dg, mirror=False)
            ops.linear_bwd_weight_sym(self.du, self.g[k], d["w1"][k])
            gm, gy = self.df, self.dy      # (the gradients of the block's result and of y_{k+1} have been read: their planes are free)
            ops.hadamard_bwd_sym(self.m[k], p["gate"][k], self.dg, gm, d["gate"][k], shared=True)
            ops.cgemm_batched(self.F, 0, ops.CMat(gm.planes[0], gm.planes[1]), S * D, ops.CMat(gy.planes[0], gy.planes[1]), S * D, S, D, S, B,
                              b_kmajor=1)
            dh = below
        ops.norm_gate_bwd_sym(self.h[0], self.s2[0], p["norm"][0], self.dy, dh, d["norm"][0], accumulate=1)
        wide = [ops.Plane(x.ptr, B, S * D, S * D) for x in dh.planes[2:]]
        ops.embedding_bwd(self.tokens, wide[0], wide[1], d["table"].planes[2], d["table"].planes[3], D, self.V, B, S)
