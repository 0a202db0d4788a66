"""The paged operators together, as a server's step: plan, store, attention and sample on a
caller's stream, captured once and replayed while the lengths grow on the device."""
import ctypes

import numpy as np
import pytest

import pitorch_amd as pa
from pitorch_amd._ffi import check
from tests import _paged as R

pytestmark = pytest.mark.gpu


class Server:
    """Device state of `S` requests and one call that enqueues a step over them."""

    def __init__(self, S, heads, kv, hd, page, kind, max_rows, max_len, vocab, seed):
        from pitorch_amd._hip import DeviceArray
        self.L, self.rng = pa.load_ptmi(), np.random.default_rng(seed)
        self.S, self.H, self.KV, self.hd, self.page, self.kind, self.R, self.V = S, heads, kv, hd, page, kind, max_rows, vocab
        self.W = R.pages_for(max_len, page)
        self.n_pages = S * self.W
        dt = np.uint16 if kind == pa.BF16 else np.float32
        n = self.n_pages * page * kv * hd
        self.k, self.v = (DeviceArray.from_host(np.full(n, 0x7FC1 if kind == pa.BF16 else np.nan).astype(dt)) for _ in range(2))
        ints = lambda n, v=0: DeviceArray.from_host(np.full(max(n, 1), v, np.int32))  # noqa: E731
        self.kv_len, self.fresh, self.count = ints(S), ints(S), ints(1, self.n_pages)
        self.pool = DeviceArray.from_host(self.rng.permutation(self.n_pages).astype(np.int32))
        self.table, self.start, self.pos, self.slot = ints(S * self.W, -1), ints(S + 1), ints(max_rows), ints(max_rows)
        self.status, self.token = ints(1), ints(S)
        a = np.arange(max_len)[:, None] * np.exp(-np.arange(0, hd, 2) * 9.21 / hd)
        self.rope_host = np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)
        self.rope = DeviceArray.from_host(self.rope_host.reshape(-1))
        self.ld = (heads + 2 * kv) * hd
        self.qkv, self.out = DeviceArray(max_rows * self.ld), DeviceArray(max_rows * heads * hd)
        self.logits, self.u = DeviceArray(S * vocab), DeviceArray(S)
        self.pages = R.pages_struct(self.k.ptr, self.v.ptr, kind, self.n_pages, page, kv, hd)
        self.nb = self.L.ptmi_paged_attention_work(R.byref(self.pages), heads, 0)
        self.work = DeviceArray(self.nb, np.uint8)
        self.host = [np.zeros((0, kv, hd), np.float32) for _ in range(2 * S)]      # keys, values by request

    def enqueue(self, stream, max_new):
        L, p = self.L, R.byref(self.pages)
        q, k, v = self.qkv.ptr, self.qkv.ptr + 4 * self.H * self.hd, self.qkv.ptr + 4 * (self.H + self.KV) * self.hd
        check(L.ptmi_paged_plan_dev(self.kv_len.ptr, self.fresh.ptr, self.S, self.pool.ptr, self.count.ptr, self.n_pages, self.page,
                                    self.table.ptr, self.W, self.kv_len.ptr, self.count.ptr, self.start.ptr, self.pos.ptr,
                                    self.slot.ptr, self.R, self.status.ptr, stream))
        check(L.ptmi_paged_store_dev(p, q, self.ld, q, self.ld, self.H, k, v, self.ld, self.pos.ptr, self.slot.ptr, self.R,
                                     self.rope.ptr, len(self.rope_host), stream))
        check(L.ptmi_paged_attention_dev(p, self.table.ptr, self.W, self.start.ptr, self.kv_len.ptr, self.S, max_new, q, self.ld,
                                         self.out.ptr, self.H * self.hd, self.R, self.H, self.hd ** -0.5, self.work.ptr, self.nb, stream))
        check(L.ptmi_sample_dev(self.logits.ptr, self.V, self.S, self.V, None, None, None, None, self.u.ptr, self.token.ptr, stream))

    def inputs(self, fresh):
        """New random rows, logits and numbers for a step."""
        self.n = list(fresh)
        self.x = self.rng.standard_normal((self.R, self.ld)).astype(np.float32)
        self.lg, self.un = self.rng.standard_normal((self.S, self.V)).astype(np.float32), self.rng.random(self.S).astype(np.float32)
        self.fresh.upload(np.array(fresh, np.int32))
        self.qkv.upload(self.x.reshape(-1))
        self.out.upload(np.full(self.R * self.H * self.hd, R.SENTINEL))
        self.logits.upload(self.lg.reshape(-1))
        self.u.upload(self.un)

    def verify(self):
        H, KV, hd = self.H, self.KV, self.hd
        assert self.status.download()[0] == 0
        lens, start = self.kv_len.download()[:self.S], self.start.download()
        out = self.out.download().reshape(self.R, H, hd)
        row = 0
        for s, n in enumerate(self.n):
            assert start[s] == row
            if n < 0:
                self.host[2 * s] = self.host[2 * s + 1] = np.zeros((0, KV, hd), np.float32)
            past = len(self.host[2 * s])
            n = max(n, 0)
            assert lens[s] == past + n
            q, k, v = np.split(self.x[row:row + n].reshape(n, H + 2 * KV, hd), [H, H + KV], 1)
            pos = np.arange(past, past + n)
            q, k = R.rotate(q, pos, self.rope_host), R.rotate(k, pos, self.rope_host)
            if self.kind == pa.BF16:
                k, v = R.from_bf16(R.bf16(k)), R.from_bf16(R.bf16(v))
            K = self.host[2 * s] = np.concatenate((self.host[2 * s], k))
            V = self.host[2 * s + 1] = np.concatenate((self.host[2 * s + 1], v))
            if n:
                page = max(len(K), 1)                        # its tokens as one page
                want = np.zeros((n, H, hd))
                bound = R.attention(q, K, V, np.zeros((1, 1), np.int64), page, 1, np.array([0, n]), np.array([len(K)]), hd ** -0.5, want)
                assert (np.abs(out[row:row + n] - want) <= bound).all(), s
            row += n
        assert start[self.S] == row and (out[row:] == R.SENTINEL).all()
        tok = self.token.download()
        for s in range(self.S):
            t, margin = R.sample(self.lg[s], u=float(self.un[s]))
            assert tok[s] == t or margin < self.V * 2.0**-44


def stream():
    from pitorch_amd._hip import hip
    p = ctypes.c_void_p()
    assert hip().hipStreamCreateWithFlags(ctypes.byref(p), 1) == 0
    return p.value


SHAPES = [dict(S=5, heads=6, kv=6, hd=48, page=16, kind=pa.F32), dict(S=3, heads=8, kv=2, hd=64, page=24, kind=pa.BF16)]


@pytest.mark.parametrize("shape", SHAPES, ids=("heads", "shared_heads"))
@pytest.mark.parametrize("unknown", [False, True])
def test_a_captured_step_serves_growing_requests(shape, unknown):
    """One graph per kind of step; eager work and synchronisation between the replays.  max_new as
    the step has it, or not known."""
    from pitorch_amd._hip import Graph, hip
    s = Server(max_rows=200, max_len=300, vocab=700, seed=3, **shape)
    st = stream()
    S = shape["S"]
    s.inputs([0] * S)
    s.enqueue(st, 0)                                         # (everything is loaded before the capture)
    assert hip().hipStreamSynchronize(st) == 0
    s.verify()
    decode = Graph(st, lambda: s.enqueue(st, 0 if unknown else 1))
    chunk = Graph(st, lambda: s.enqueue(st, 0))
    steps = [([70, 0, 1, 33, 90][:S], chunk)] + [([1, 0, 1, 1, 1][:S], decode)] * 3 + [([2, 60, 40, -1, 1][:S], chunk)] + \
        [([1, 1, 1, 0, 1][:S], decode), ([-1, 5, 1, 40, 0][:S], chunk), ([30, 0, 1, 1, 1][:S], chunk)] + [([1] * S, decode)] * 2
    for i, (fresh, graph) in enumerate(steps):
        s.inputs(fresh)
        graph.launch()
        assert hip().hipStreamSynchronize(st) == 0
        s.verify()
        if i % 3 == 1:                                       # an eager step in between
            s.inputs([1] * S)
            s.enqueue(st, 1)
            assert hip().hipStreamSynchronize(st) == 0
            s.verify()
    decode.free()
    chunk.free()
    hip().hipStreamDestroy(st)


def test_two_servers_at_once():
    """Two captured steps on two streams, each with its own workspace, in flight together."""
    from pitorch_amd._hip import Graph, hip
    servers = [Server(max_rows=64, max_len=400, vocab=500, seed=i, **SHAPES[i]) for i in range(2)]
    streams = [stream() for _ in servers]
    for s, st in zip(servers, streams):
        s.inputs([60 // s.S] * s.S)
        s.enqueue(st, 0)
    for s, st in zip(servers, streams):
        assert hip().hipStreamSynchronize(st) == 0
        s.verify()
    graphs = [Graph(st, lambda s=s, st=st: s.enqueue(st, 0)) for s, st in zip(servers, streams)]
    for i in range(6):
        for s in servers:
            s.inputs([1 + (i + j) % 3 * (i % 2) * 5 for j in range(s.S)])
        for g in graphs:
            g.launch()
        for st in streams:
            assert hip().hipStreamSynchronize(st) == 0
        for s in servers:
            s.verify()
    for g, st in zip(graphs, streams):
        g.free()
        hip().hipStreamDestroy(st)


def test_a_refused_step_does_nothing():
    """More rows than there is room for: no row has a slot, nothing is stored, no row is computed."""
    s = Server(max_rows=20, max_len=100, vocab=300, seed=5, **SHAPES[0])
    s.inputs([4] * 5)
    s.enqueue(None, 4)
    check(s.L.ptmi_sync())
    s.verify()
    before = [a.download() for a in (s.k, s.v, s.kv_len, s.count, s.table)]
    s.inputs([5] * 5)
    s.enqueue(None, 5)
    check(s.L.ptmi_sync())
    assert s.status.download()[0] == 4
    for a, b in zip((s.k, s.v, s.kv_len, s.count, s.table), before):
        assert np.array_equal(a.download().view(np.uint8), b.view(np.uint8))
    assert (s.out.download() == R.SENTINEL).all()
    s.inputs([1] * 5)                                        # and the next step goes on
    s.enqueue(None, 1)
    check(s.L.ptmi_sync())
    s.verify()
