"""A served decode step made of the paged cache, the microscaled products and
the logits' rules together: prompts' keys and values into the pages, then steps
whose picks are the next inputs, eagerly and as a captured graph.

Every stage is compared with its definition over what the stage before it left
on the device (a rounding before a quantization may move a code, so errors are
not followed through), with the bars of the operators' own tests.
"""
import math

import numpy as np
import pytest

from tests.test_gpu_logits import same
from tests.test_gpu_logits import want as want_logits
from tests.test_gpu_mx4 import bar, quant, values
from tests.test_gpu_paged import held
from tests.test_gpu_paged import want as want_attention

pytestmark = pytest.mark.gpu

F = np.float32
LAYERS, C, HEADS, KV, HD, V, PAGE, HIST = 2, 512, 8, 2, 64, 1000, 64, 24
QKV = (HEADS + 2 * KV) * HD
PROMPTS = [70, 1, 130, 63, 0, 37]  # the fifth row is padding


class Server:
    def __init__(self, gpu, kind):
        self.torch, self.lm, self.ctx = torch, lm, ctx = gpu
        rng = np.random.default_rng(3)
        d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        w = lambda n, k: rng.normal(0, 1 / math.sqrt(k), (n, k)).astype(F)  # noqa: E731
        self.wq, self.wo = [w(QKV, C) for _ in range(LAYERS)], [w(C, HEADS * HD) for _ in range(LAYERS)]
        self.wh = w(V, C)
        self.bq = rng.normal(0, 0.1, QKV).astype(F)
        self.emb = d(rng.normal(0, 1, (V, C)).astype(F))
        mat = lambda a: lm.HipMX4Matrix.from_f32(ctx, a, reduce_rows=False)  # noqa: E731
        self.mq, self.mo, self.mh = [mat(a) for a in self.wq], [mat(a) for a in self.wo], mat(self.wh)
        self.dbq = d(self.bq)
        R = self.rows = len(PROMPTS)
        width = 4
        table = rng.permutation(R * width).reshape(R, width).astype(np.int32)
        self.table, self.kind = d(table), kind
        self.cache = lm.PagedKV(ctx, LAYERS, R * width, PAGE, KV, HD, kind)
        z = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
        self.x = [z(R, C) for _ in range(LAYERS + 1)]
        self.qkv, self.att, self.out = ([z(R, n) for _ in range(LAYERS)] for n in (QKV, HEADS * HD, C))
        self.codes = [z(R, C // 2, t=torch.uint8) for _ in range(2 * LAYERS + 1)]
        self.scales = [z(R, C // 32, t=torch.uint8) for _ in range(2 * LAYERS + 1)]
        self.logits, self.adjusted = z(R, V), z(R, V)
        self.tok, self.pick = z(R, t=torch.int64), z(R, t=torch.int64)
        self.work = z(self.cache.work_bytes(R, HEADS), t=torch.uint8)
        self.lwork = z(lm.logits_work_bytes(R, V), t=torch.uint8)
        self.hist = torch.full((R, HIST), -1, dtype=torch.int32, device="cuda")  # -1: no token yet
        self.count = z(R, t=torch.int64)
        self.hoff = d((np.arange(R + 1) * HIST).astype(np.int64))
        self.rep, self.freq = d(rng.uniform(1, 1.5, R).astype(F)), d(rng.uniform(0, 0.5, R).astype(F))
        self.mask = d(rng.integers(-2 ** 31, 2 ** 31, (R, -(-V // 32))).astype(np.int32))
        # prompts
        seq = np.concatenate([np.full(n, r, np.int32) for r, n in enumerate(PROMPTS)])
        pos = np.concatenate([np.arange(n, dtype=np.int32) for n in PROMPTS])
        x = self.emb[d(rng.integers(0, V, len(seq)))]
        for l in range(LAYERS):
            y = z(len(seq), QKV)
            lm.linear(ctx, y, x, self.mq[l], self.dbq)
            k, v = self.split(y)[1:]
            self.cache.store(l, k, v, d(seq), d(pos), self.table)
        self.pos = d(np.array([n if n else -1 for n in PROMPTS], np.int32))
        self.tok.copy_(d(rng.integers(0, V, R)))

    @staticmethod
    def split(y):
        q, k, v = y.split([HEADS * HD, KV * HD, KV * HD], 1)
        return q.unflatten(1, (HEADS, HD)), k.unflatten(1, (KV, HD)), v.unflatten(1, (KV, HD))

    def step(self):
        torch, lm, ctx = self.torch, self.lm, self.ctx

        def product(i, out, x, m, **kw):
            lm.mx4_quantize(ctx, x, self.codes[i], self.scales[i])
            lm.mx4_linear(ctx, out, self.codes[i], self.scales[i], m, **kw)

        torch.index_select(self.emb, 0, self.tok, out=self.x[0])
        for l in range(LAYERS):
            product(2 * l, self.qkv[l], self.x[l], self.mq[l], bias=self.dbq)
            q, k, v = self.split(self.qkv[l])
            self.cache.step(l, self.att[l], q, k, v, self.pos, self.table, self.work, cap=20.0)
            self.x[l + 1].copy_(self.x[l])
            product(2 * l + 1, self.x[l + 1], self.att[l], self.mo[l], resid=True)
        product(2 * LAYERS, self.logits, self.x[LAYERS], self.mh)
        lm.adjust_logits(ctx, self.adjusted, self.logits, history=(self.hist.view(-1), self.hoff), repetition=self.rep,
                         frequency=self.freq, mask=self.mask, pick=self.pick, work=self.lwork)
        self.tok.copy_(self.pick)
        self.hist.scatter_(1, self.count[:, None], self.pick[:, None].int())
        self.count += 1
        self.pos += (self.pos >= 0).int()

    def check(self, pos, hist):
        """The step just done, from positions pos and histories hist."""
        torch = self.torch
        n = lambda t: t.cpu().numpy()  # noqa: E731

        def operand(i, x):
            c, s = n(self.codes[i]), n(self.scales[i])
            qc, qs = quant(x)
            assert np.array_equal(c, qc) and np.array_equal(s, qs)
            return values(c, s)

        for l in range(LAYERS):
            x, w = operand(2 * l, n(self.x[l])), values(*quant(self.wq[l]))
            y = x @ w.T + self.bq
            assert np.all(np.abs(n(self.qkv[l]) - y) <= bar(x, w, self.bq) + 2.0 ** -24 * np.abs(y))
            q, k, v = (n(t) for t in self.split(self.qkv[l]))
            got = n(self.att[l]).reshape(-1, HEADS, HD)
            for r, p in enumerate(pos):
                if p < 0:
                    assert np.all(got[r] == 0)
                    continue
                at = [torch.full((p + 1,), r, dtype=torch.int32, device="cuda"),
                      torch.arange(p + 1, dtype=torch.int32, device="cuda")]
                fk, fv = (torch.empty(p + 1, KV, HD, device="cuda") for _ in range(2))
                self.cache.fetch(l, fk, fv, *at, self.table)
                fk, fv = n(fk), n(fv)
                assert np.array_equal(fk[p], held(self.kind, k[r])) and np.array_equal(fv[p], held(self.kind, v[r]))
                o, b = want_attention(q[r], fk, fv, 1 / math.sqrt(HD), 20.0, None)
                assert np.all(np.abs(got[r] - o) <= b), (l, r)
            x, w, r = operand(2 * l + 1, n(self.att[l])), values(*quant(self.wo[l])), n(self.x[l])
            y = x @ w.T
            assert np.all(np.abs(n(self.x[l + 1]) - (y + r)) <= bar(x, w) + 2.0 ** -23 * (np.abs(y) + np.abs(r)))
        x, w = operand(2 * LAYERS, n(self.x[LAYERS])), values(*quant(self.wh))
        logits = n(self.logits)
        assert np.all(np.abs(logits - x @ w.T) <= bar(x, w))
        o, p = want_logits(logits, hist=hist.reshape(-1), hoff=n(self.hoff), rep=n(self.rep), freq=n(self.freq),
                           mask=n(self.mask))
        assert same(n(self.adjusted), o) and np.array_equal(n(self.pick), p)


@pytest.mark.parametrize("kind", ["int8", "f16"])
def test_steps(gpu, kind):
    torch, lm, ctx = gpu
    a, b = Server(gpu, kind), Server(gpu, kind)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin()
            b.step()
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in range(6):
        pos, hist = a.pos.cpu().numpy(), a.hist.cpu().numpy()
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        a.check(pos, hist)
        for s, t in ((a.x[LAYERS], b.x[LAYERS]), (a.adjusted, b.adjusted), (a.pick, b.pick), (a.pos, b.pos)):
            assert torch.equal(s, t), i


def test_two_graphs_at_once(gpu):
    """Two servers' captured steps side by side on two streams, each with its
    own workspaces, equal one after another."""
    torch, lm, ctx = gpu
    servers = [Server(gpu, "int8") for _ in range(3)]
    servers[1].tok += 5
    servers[2].tok += 5
    servers[1].tok %= V
    servers[2].tok %= V
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    for s, st, g in zip(servers, streams, graphs):
        try:
            with torch.cuda.stream(st):
                ctx.set_stream(st)
                g.capture_begin()
                s.step()
                g.capture_end()
        finally:
            ctx.set_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    alone = Server(gpu, "int8")
    for i in range(8):
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        alone.step()
        servers[2].step()
        torch.cuda.synchronize()
        assert torch.equal(servers[0].adjusted, alone.adjusted) and torch.equal(servers[0].pick, alone.pick), i
        assert torch.equal(servers[1].adjusted, servers[2].adjusted), i
        assert torch.equal(servers[1].pick, servers[2].pick), i
