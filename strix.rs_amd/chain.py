"""The FFN half of a decoder stack as a sequence of resident, device-routed calls: what an orchestrator captures once
as a HIP graph and replays per token (the reference's captured token, crates/strix-backend-rocm/src/decode.rs:3053-3203,
and its per-layer launch sequence, decode.rs:1136-1180: router logits -> topk_router -> moe_launches).

Per layer, four calls / five launches:
    1. smx_ffn_gate_up_dev     rmsnorm + quantiser + gate and up GEMVs + SwiGLU product   x -> h[ffn]
    2. smx_gemv_dev            quantiser + down GEMV                                      h -> d[hidden]
    3. smx_gemv_dev            router logits GEMV                                         d -> logits[ne]
    4. smx_moe_ffn_logits_dev  softmax + top-k in the prologue of the k routed experts' gate/up launch, then their down
                               launch                                                     d, logits -> y[hidden] (+ ids[k], w[k])
(route="call": the router as smx_moe_router_dev, route="launches": as smx_gemv_dev + smx_moe_route_dev, each followed by
smx_moe_ffn_routed_dev: six launches, same bits.)
The benchmark (bench.py) and the parity test (tests/test_gpu_chain.py) both run this class, so what is measured is what is checked.

AttentionChain is the other half, for a batch of sequences: projections, the paged cache and the attention over it, and the sampled
token at the end (the reference's rope, append and sdpa of decode.rs:1136-1180, 5326-5368).  tests/test_gpu_attention_chain.py runs it.
"""


class FfnMoeChain:
    """keys(l) -> (gate, up, down, router) weight keys of layer l; moe_layer(l) -> resident MoE layer index.

    keep_stages: every layer gets buffers of its own for h, d, logits, ids, w and y, so that a test can read each stage back;
    otherwise the layers share one set (what a decode loop does)."""

    def __init__(self, acc, layers, hidden, ffn, ne, k, keys, moe_layer, norm_w_dev, eps=1e-6, keep_stages=False,
                 route="in_launch"):
        self.acc, self.layers, self.hidden, self.ffn, self.ne, self.k = acc, layers, hidden, ffn, ne, k
        self.keys, self.moe_layer, self.norm_w_dev, self.eps = keys, moe_layer, norm_w_dev, eps
        assert route in ("in_launch", "call", "launches")
        self.route = route
        self._bufs = []
        nsets = layers if keep_stages else 1
        self.stage = []
        for _ in range(nsets):
            b = {"h": self._alloc(ffn * 4), "d": self._alloc(hidden * 4), "logits": self._alloc(ne * 4),
                 "ids": self._alloc(k * 4), "w": self._alloc(k * 4)}
            self.stage.append(b)
        # layer outputs alternate between two buffers (a layer reads the previous layer's output); with keep_stages each its own
        self.y = [self._alloc(hidden * 4) for _ in range(layers if keep_stages else 2)]

    def _alloc(self, nbytes):
        p = self.acc.dev_alloc(nbytes)
        self._bufs.append(p)
        return p

    def buffers(self, l):
        """(stage buffers, output buffer) of layer l."""
        return self.stage[l % len(self.stage)], self.y[l % len(self.y)]

    def enqueue(self, x_dev, layer_offset=0):
        """Enqueue all layers on the context's stream (capturable); returns the device buffer holding the last layer's output.
        layer_offset: added to the layer index when naming weights (rotating weight sets of a benchmark)."""
        acc, cur = self.acc, x_dev
        for l in range(self.layers):
            b, y = self.buffers(l)
            gate, up, down, router = self.keys(l + layer_offset)
            ok = acc.ffn_gate_up_dev(gate, up, 2, cur, b["h"], norm=True, norm_w_dev=self.norm_w_dev, eps=self.eps)
            ok = ok and acc.gemv_dev(down, b["h"], 1, b["d"])
            layer = self.moe_layer(l + layer_offset)
            if self.route == "in_launch":
                ok = ok and acc.gemv_dev(router, b["d"], 1, b["logits"])
                ok = ok and acc.moe_ffn_logits_dev(layer, b["logits"], self.k, b["d"], y, b["ids"], b["w"])
            else:
                if self.route == "call":
                    ok = ok and acc.moe_router_dev(router, b["d"], self.k, b["ids"], b["w"], b["logits"])
                else:
                    ok = ok and acc.gemv_dev(router, b["d"], 1, b["logits"])
                    ok = ok and acc.moe_route_dev(b["logits"], self.ne, self.k, b["ids"], b["w"])
                ok = ok and acc.moe_ffn_routed_dev(layer, b["ids"], b["w"], self.k, b["d"], y)
            if not ok:
                raise RuntimeError(f"layer {l}: a weight of the chain is not resident")
            cur = y
        return cur

    def launches_per_token(self):
        """(when the experts' gate/up launch routes: up to 64 experts, k <= 8, flat-form expert rows)"""
        return self.layers * (5 if self.route == "in_launch" else 6)

    def close(self):
        for p in self._bufs:
            self.acc.dev_free(p)
        self._bufs = []


class AttentionChain:
    """The attention half of a decoder stack and the sampled end of a step, for a batch of sequences over paged 8-bit caches.

    Per layer:
        1. rmsnorm + quantiser + q, k and v projections  x -> q, k, v   (one row: one launch; more: a launch and a GEMM each)
        2. smx_kv_append_dev   q and k rotated, k and v into the layer's cache
        3. smx_attn_dev        q over the cache -> o
        4. smx_gemv_dev        quantiser + output projection            o -> y[hidden]
    and behind the last layer rmsnorm + lm_head and smx_sample_dev on the rows that the caller names.  enqueue() runs one layer's output straight
    into the next; a caller with something of its own between them (a residual, the other half of the layer) calls layer() for each.

    Each call's rows, lengths and page table are a KvBatch of the caller's, whose device arrays the kernels read when they run: a
    captured decode step (one row for each sequence) serves every later one, with new lengths and pages written in front of it.

    pkg: the package module (its KvCache, KvBatch and Rope); keys(l) -> (q, k, v, o) weight keys of layer l; norm_w_dev: the rmsnorm weight
    of every layer and of the end, or a list of layers + 1 of them; rows: the most that one call brings.  keep_stages: every layer gets
    buffers of its own, so that a test can read each stage back."""

    def __init__(self, pkg, acc, layers, hidden, q_heads, kv_heads, head_dim, keys, lm_head, vocab, norm_w_dev, rows, pages, page_tokens, max_pos,
                 rope_base=1e4, window=0, eps=1e-6, keep_stages=False):
        self.pkg, self.acc, self.layers, self.hidden, self.keys = pkg, acc, layers, hidden, keys
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.lm_head, self.vocab, self.rows, self.window, self.eps = lm_head, vocab, rows, window, eps
        self.norms = list(norm_w_dev) if isinstance(norm_w_dev, (list, tuple)) else [norm_w_dev] * (layers + 1)
        if len(self.norms) != layers + 1:
            raise ValueError(f"{len(self.norms)} rmsnorm weights for {layers} layers and the end")
        self._bufs = []
        code_bytes, scales = pkg.kv_sizes(pages, page_tokens, kv_heads, head_dim)
        self.cache = [pkg.KvCache(pages, page_tokens, kv_heads, head_dim, self._alloc(code_bytes), self._alloc(code_bytes), self._alloc(scales * 4),
                                  self._alloc(scales * 4)) for _ in range(layers)]
        table = self._alloc(max_pos * head_dim * 4)
        acc.rope_table_dev(rope_base, head_dim, max_pos, table)
        self.rope = pkg.Rope(table, max_pos, head_dim)
        qw, kw = rows * q_heads * head_dim * 4, rows * kv_heads * head_dim * 4
        self.stage = [{"q": self._alloc(qw), "k": self._alloc(kw), "v": self._alloc(kw), "o": self._alloc(qw)} for _ in range(layers if keep_stages else 1)]
        self.y = [self._alloc(rows * hidden * 4) for _ in range(layers if keep_stages else 2)]
        self.logits = self._alloc(rows * vocab * 4)

    def _alloc(self, nbytes):
        p = self.acc.dev_alloc(nbytes)
        self._bufs.append(p)
        return p

    def buffers(self, l):
        """(stage buffers, output buffer) of layer l."""
        return self.stage[l % len(self.stage)], self.y[l % len(self.y)]

    def _fits(self, rows):
        if rows > self.rows:
            raise ValueError(f"{rows} rows, buffers for {self.rows}")

    def _project(self, keys, x_dev, norm_w, rows, outs):
        """rmsnorm of rows of x_dev through the projections `keys`."""
        if rows == 1:
            return self.acc.gemv_fused_dev(list(keys), self.pkg.ACT_RMSNORM, x_dev, norm_w, list(outs), self.eps)
        return all([self.acc.gemm_fused_dev(k, self.pkg.ACT_RMSNORM, x_dev, norm_w, rows, y, self.eps) for k, y in zip(keys, outs)])

    def layer(self, l, x_dev, batch):
        """Enqueue layer l for the rows of `batch`; returns the device buffer holding its output."""
        self._fits(batch.rows)
        acc, (b, y), (q, k, v, o) = self.acc, self.buffers(l), self.keys(l)
        ok = self._project((q, k, v), x_dev, self.norms[l], batch.rows, (b["q"], b["k"], b["v"]))
        if ok:
            acc.kv_append_dev(self.cache[l], batch, b["k"], b["v"], rope=self.rope, q=b["q"], q_heads=self.q_heads, q_out=b["q"])
            acc.attn_dev(self.cache[l], batch, b["q"], self.q_heads, self.head_dim ** -0.5, b["o"], window=self.window)
            ok = (acc.gemv_dev if batch.rows <= 32 else acc.gemm_dev)(o, b["o"], batch.rows, y)
        if not ok:
            raise RuntimeError(f"layer {l}: a weight of the chain is not resident")
        return y

    def enqueue(self, x_dev, batch):
        """Enqueue all layers for the rows of `batch` on the context's stream (capturable once a call of the same sizes has run); returns the
        device buffer holding the last layer's output."""
        cur = x_dev
        for l in range(self.layers):
            cur = self.layer(l, cur, batch)
        return cur

    def sample(self, y_dev, rows, u_dev, ids_dev, temperature=None, top_k=None, top_p=None, min_p=None, prob=None):
        """Enqueue rmsnorm, the lm_head and the pick of one token for each of `rows` rows of hidden states (device arrays throughout)."""
        self._fits(rows)
        if not self._project((self.lm_head,), y_dev, self.norms[-1], rows, (self.logits,)):
            raise RuntimeError("the lm_head is not resident")
        self.acc.sample_dev(self.logits, rows, self.vocab, u_dev, ids_dev, temperature, top_k, top_p, min_p, prob)

    def close(self):
        self.acc.sync()
        for p in self._bufs:
            self.acc.dev_free(p)
        self._bufs = []
