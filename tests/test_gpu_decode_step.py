"""A batch that shares a prompt, decoded step by step as a program would: the e4m3 projections, rotary
positions with the store into a paged cache, attention over the prompt and each sequence's own keys, and
the adjusted logits that softmax and argmax go by. Every call of every step is held to its 64-bit form on
what the device had; then the same calls recorded into graphs and replayed."""
import ctypes as C
import threading

import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import assert_within, csr, dev, logits_adjust, narrow, packed, ptr, rope, rounding, sdpa_prefix, widen
from hipmem import DevBuf, check, hip as hiprt, synchronize
from kurumi_amd import DType, Graph, Tensor
from test_gpu_linear_e4m3 import quantise_rows

pytestmark = pytest.mark.gpu
DT = DType.BF16


def put(buf: DevBuf, a: np.ndarray) -> None:
    a = np.ascontiguousarray(a)
    check(hiprt().hipMemcpy(buf.ptr, a.ctypes.data, a.nbytes, 1), "hipMemcpy H2D")


class Layer:
    """One attention layer and the output head on the device, with its caches."""

    def __init__(self, nb=3, hidden=256, heads=4, kv=2, d=64, prompt=45, page=8, vocab=1003, history=64, seed=1):
        self.nb, self.hidden, self.heads, self.kv, self.d, self.prompt, self.page, self.vocab, self.history = nb, hidden, heads, kv, d, prompt, page, vocab, history
        rng = self.rng = np.random.default_rng(seed)
        self.row = (heads + 2 * kv) * d
        self.weights = {}
        for name, n, k in (("qkv", self.row, hidden), ("out", hidden, heads * d), ("head", vocab, hidden)):
            wq, sw = quantise_rows((rng.standard_normal((n, k)) * 0.06).astype(np.float32))
            self.weights[name] = (dev(wq), dev(sw), n, k)
        self.per_seq = 6
        self.pages = rng.permutation(nb * self.per_seq + 3)[: nb * self.per_seq].reshape(nb, self.per_seq).astype(np.int32)
        self.rows = (nb * self.per_seq + 3) * page
        self.freqs = K.rope_freqs(d, 10000.0, K.ROPE_BY_PARTS, factor=4.0, trained_len=64.0)
        z = lambda n, dt=np.uint16: dev(np.zeros(n, dt))  # noqa: E731
        self.x, self.qkv, self.att, self.y = z(nb * hidden), z(nb * self.row), z(nb * heads * d), z(nb * hidden)
        self.logits, self.adjusted = z(nb * vocab), z(nb * vocab, np.float32)
        self.pk, self.pv = z(prompt * kv * d), z(prompt * kv * d)
        self.ck, self.cv = z(self.rows * kv * d), z(self.rows * kv * d)
        self.dpages, self.positions, self.slots, self.lens = dev(self.pages), z(nb, np.int32), z(nb, np.int32), z(nb, np.int32)
        self.tokens, self.nlens, self.nprompt = z((nb, history), np.int32), z(nb, np.int32), z(nb, np.int32)
        self.rep, self.pres, self.freq = (dev(np.full(nb, v, np.float32)) for v in (1.3, 0.4, 0.2))
        self.bias = [[(5, 3.0), (7 + b, -2.0)] for b in range(nb)]
        self.dbias = [dev(x) for x in csr(self.bias)]
        self.mask = rng.random((2, vocab)) < 0.7
        self.dmask, self.index = dev(packed(self.mask)), np.array([0, -1, 1][:nb], np.int32)
        self.dindex = dev(self.index)
        self.rope_args = K.RopeArgs(
            dtype=DT, layout=K.ROPE_HALF, scale=1.0, tokens=nb, q_heads=heads, kv_heads=kv, head_dim=d, rot_dim=d, freqs=self.freqs,
            positions=self.positions.ptr, q=self.qkv.ptr, q_token_stride=self.row, q_head_stride=d, q_out=self.qkv.ptr, q_out_token_stride=self.row,
            q_out_head_stride=d, k=ptr(self.qkv, heads * d, DT), k_token_stride=self.row, k_head_stride=d, k_out=self.ck.ptr, k_out_row_stride=kv * d,
            k_out_head_stride=d, v=ptr(self.qkv, (heads + kv) * d, DT), v_token_stride=self.row, v_head_stride=d, v_out=self.cv.ptr,
            v_out_row_stride=kv * d, v_out_head_stride=d, rows=self.slots.ptr, out_rows=self.rows)
        self.sdpa_args = K.SdpaPrefixArgs(
            dtype=DT, scale=1 / np.sqrt(d), batch=nb, q_len=1, q_heads=heads, kv_heads=kv, head_dim=d, q=self.qkv.ptr, q_batch_stride=self.row,
            q_token_stride=self.row, q_head_stride=d, out=self.att.ptr, out_batch_stride=heads * d, out_token_stride=heads * d, out_head_stride=d,
            prefix_len=prompt, prefix_k=self.pk.ptr, prefix_v=self.pv.ptr, prefix_row_stride=kv * d, prefix_head_stride=d,
            own_max=self.per_seq * page, own_lens=self.lens.ptr, own_k=self.ck.ptr, own_v=self.cv.ptr, own_row_stride=kv * d, own_head_stride=d,
            own_rows=self.rows, pages=self.dpages.ptr, page_size=page, pages_per_seq=self.per_seq)
        self.logits_args = K.LogitsArgs(
            dtype=DT, out_dtype=DType.F32, rows=nb, vocab=vocab, logits=self.logits.ptr, logits_stride=vocab, out=self.adjusted.ptr,
            out_stride=vocab, history=history, tokens=self.tokens.ptr, tokens_stride=history, lens=self.nlens.ptr, prompt_lens=self.nprompt.ptr,
            repetition=self.rep.ptr, presence=self.pres.ptr, frequency=self.freq.ptr, bias_ids=self.dbias[0].ptr, bias_values=self.dbias[1].ptr,
            bias_offsets=self.dbias[2].ptr, bias_count=2 * nb, mask=self.dmask.ptr, mask_rows=2, mask_stride=-(-vocab // 32), mask_index=self.dindex.ptr)
        self.scratch = DevBuf(K.sdpa_prefix_scratch(self.sdpa_args))
        self.step = 0
        self.history_np = rng.integers(0, vocab, (nb, history)).astype(np.int32)

    def linear(self, hip, name, x, y, m):
        wq, sw, n, k = self.weights[name]
        hip.linear_e4m3(x.ptr, DT, wq.ptr, sw.ptr, y.ptr, DT, m, n, k)

    def prefill(self, hip):
        """The prompt's keys and values, rotated, in their own rows."""
        x, qkv = dev(narrow(self.rng.standard_normal((self.prompt, self.hidden)), DT)), DevBuf(self.prompt * self.row * 2)
        self.linear(hip, "qkv", x, qkv, self.prompt)
        pos = dev(np.arange(self.prompt, dtype=np.int32))
        h, kv, d = self.heads, self.kv, self.d
        hip.rope(K.RopeArgs(dtype=DT, layout=K.ROPE_HALF, scale=1.0, tokens=self.prompt, kv_heads=kv, head_dim=d, rot_dim=d, freqs=self.freqs,
                            positions=pos.ptr, k=ptr(qkv, h * d, DT), k_token_stride=self.row, k_head_stride=d, k_out=self.pk.ptr,
                            k_out_row_stride=kv * d, k_out_head_stride=d, v=ptr(qkv, (h + kv) * d, DT), v_token_stride=self.row, v_head_stride=d,
                            v_out=self.pv.ptr, v_out_row_stride=kv * d, v_out_head_stride=d, out_rows=self.prompt))
        synchronize()
        bits = qkv.numpy(np.uint16, (self.prompt, self.row))[:, h * d :].reshape(self.prompt, 2 * kv, d)
        want, tol = rope(widen(bits[:, :kv], DT), np.arange(self.prompt), list(self.freqs), d, K.ROPE_HALF)
        assert_within(widen(self.pk.numpy(np.uint16, (self.prompt, kv, d)), DT), want, tol + rounding(want, DT), "prompt keys")
        np.testing.assert_array_equal(self.pv.numpy(np.uint16, (self.prompt, kv, d)), bits[:, kv:])

    def place(self):
        """The new token's position, cache row and lengths; sequence b has b tokens more than sequence 0."""
        n = self.step + np.arange(self.nb)
        put(self.positions, (self.prompt + n).astype(np.int32))
        put(self.slots, (self.pages[np.arange(self.nb), n // self.page] * self.page + n % self.page).astype(np.int32))
        put(self.lens, (n + 1).astype(np.int32))
        put(self.tokens, self.history_np)
        put(self.nlens, np.full(self.nb, 20 + self.step, np.int32))
        put(self.nprompt, np.full(self.nb, 9, np.int32))
        self.step += 1
        return n

    def calls(self, hip, stream=None, scratch=True):
        """The layer's three calls between its projections."""
        self.sdpa_args.scratch, self.sdpa_args.scratch_bytes = (self.scratch.ptr, self.scratch.nbytes) if scratch else (None, 0)
        hip.rope(self.rope_args, stream)
        hip.sdpa_prefix(self.sdpa_args, stream)
        hip.logits_adjust(self.logits_args, stream)

    def state(self):
        synchronize()
        nb, kv, d = self.nb, self.kv, self.d
        return dict(qkv=self.qkv.numpy(np.uint16, (nb, self.row)), ck=self.ck.numpy(np.uint16, (self.rows, kv, d)),
                    cv=self.cv.numpy(np.uint16, (self.rows, kv, d)), att=self.att.numpy(np.uint16, (nb, 1, self.heads, d)),
                    logits=self.logits.numpy(np.uint16, (nb, self.vocab)), adjusted=self.adjusted.numpy(np.float32, (nb, self.vocab)))

    def check(self, before, after, n):
        """`after` the three calls on the qkv and caches of `before`, for tokens at own positions n."""
        h, kv, d = self.heads, self.kv, self.d
        x = widen(before["qkv"], DT).reshape(self.nb, h + 2 * kv, d)
        want, tol = rope(x[:, : h + kv], self.prompt + n, list(self.freqs), d, K.ROPE_HALF)
        slots = self.pages[np.arange(self.nb), n // self.page] * self.page + n % self.page
        got = widen(after["qkv"], DT).reshape(x.shape)
        assert_within(got[:, :h], want[:, :h], (tol + rounding(want, DT))[:, :h], "queries")
        assert_within(widen(after["ck"], DT)[slots], want[:, h:], (tol + rounding(want, DT))[:, h:], "stored keys")
        np.testing.assert_array_equal(after["cv"][slots], before["qkv"].reshape(self.nb, -1, d)[:, h + kv :])
        rest = np.setdiff1d(np.arange(self.rows), slots)
        np.testing.assert_array_equal(after["ck"][rest], before["ck"][rest])
        np.testing.assert_array_equal(after["cv"][rest], before["cv"][rest])
        w = lambda b: widen(b.numpy(np.uint16, (self.prompt, kv, d)), DT)  # noqa: E731
        o, _, to, _ = sdpa_prefix(got[:, None, :h], w(self.pk), w(self.pv), widen(after["ck"], DT), widen(after["cv"], DT), n + 1,
                                  float(np.float32(1 / np.sqrt(d))), pages=self.pages, page=self.page, npages=self.rows // self.page, dt=DT)
        assert_within(widen(after["att"], DT), o, to, "attention")
        want, tol = logits_adjust(widen(after["logits"], DT), tokens=self.history_np, lens=np.full(self.nb, 19 + self.step),
                                  prompts=np.full(self.nb, 9), rep=np.full(self.nb, np.float32(1.3)), pres=np.full(self.nb, np.float32(0.4)),
                                  freq=np.full(self.nb, np.float32(0.2)), bias=self.bias, mask=self.mask, mask_index=self.index)
        assert_within(after["adjusted"], want, tol, "adjusted logits")


def test_a_batch_decoded_step_by_step(hip):
    m = Layer()
    m.prefill(hip)
    g = Graph()
    node = g.input([m.nb, m.vocab], DType.F32)
    probs = g.softmax(node, 1)
    roots = [probs, g.cast(g.argmax(probs, 1), DType.I32)]
    for step in range(11):  # past the first page
        print(f"decode step {step}", flush=True)
        put(m.x, narrow(m.rng.standard_normal((m.nb, m.hidden)), DT))
        n = m.place()
        m.linear(hip, "qkv", m.x, m.qkv, m.nb)
        before = m.state()
        hip.rope(m.rope_args)
        hip.sdpa_prefix(m.sdpa_args)
        m.linear(hip, "out", m.att, m.y, m.nb)
        m.linear(hip, "head", m.y, m.logits, m.nb)
        hip.logits_adjust(m.logits_args)
        after = m.state()
        m.check(before, after, n)
        p, ids = hip.eval_many_with(g, roots, {node: Tensor.from_numpy(after["adjusted"])})
        np.testing.assert_array_equal(ids.numpy(), after["adjusted"].argmax(1))
        assert (p.numpy()[~np.isfinite(after["adjusted"])] == 0).all()
        m.history_np[:, 20 + step] = ids.numpy()  # the generated token joins the history


class Recorded:
    """Calls recorded from a stream into a graph."""

    def __init__(self, calls):
        L, self.stream, graph, self.exe = hiprt(), C.c_void_p(), C.c_void_p(), C.c_void_p()
        check(L.hipStreamCreate(C.byref(self.stream)), "hipStreamCreate")
        check(L.hipStreamBeginCapture(self.stream, 1), "hipStreamBeginCapture")
        self.error = None
        try:
            calls(self.stream.value)
        except K.KuError as e:
            self.error = str(e)
        check(L.hipStreamEndCapture(self.stream, C.byref(graph)), "hipStreamEndCapture")
        if self.error is None:
            check(L.hipGraphInstantiate(C.byref(self.exe), graph, None, None, C.c_size_t(0)), "hipGraphInstantiate")
        check(L.hipGraphDestroy(graph), "hipGraphDestroy")

    def replay(self):
        check(hiprt().hipGraphLaunch(self.exe, self.stream), "hipGraphLaunch")
        check(hiprt().hipStreamSynchronize(self.stream), "hipStreamSynchronize")

    def close(self):
        if self.exe:
            check(hiprt().hipGraphExecDestroy(self.exe), "hipGraphExecDestroy")
        check(hiprt().hipStreamDestroy(self.stream), "hipStreamDestroy")


def test_two_recorded_graphs_replayed_between_eager_work(hip):
    """Two layers' calls, recorded with a scratch each, replayed by turns with new inputs, with eager calls
    that grow the backend's workspace in between: every replay equals the eager calls on the same inputs."""
    layers = [Layer(seed=1), Layer(nb=2, prompt=300, seed=2)]
    for m in layers:
        m.prefill(hip)
        m.calls(hip)  # the library has seen the sizes
    graphs = [Recorded(lambda s, m=m: m.calls(hip, s)) for m in layers]
    assert all(r.error is None for r in graphs), [r.error for r in graphs]
    big = Layer(nb=3, prompt=2000, seed=3)
    for turn in range(4):
        print(f"replay {turn}", flush=True)
        starts = []
        for m in layers:
            n = m.place()
            put(m.qkv, narrow(m.rng.standard_normal((m.nb, m.row)), DT))
            put(m.logits, narrow(m.rng.standard_normal((m.nb, m.vocab)) * 3, DT))
            starts.append((n, m.state()))
        for r in graphs:
            r.replay()
        replayed = [m.state() for m in layers]
        big.place()
        big.calls(hip, scratch=False)  # eager work on the backend's workspace, larger than the graphs'
        for m, (n, before), after in zip(layers, starts, replayed):
            m.check(before, after, n)
            put(m.qkv, before["qkv"])
            put(m.ck, before["ck"])
            put(m.cv, before["cv"])
            m.calls(hip, scratch=turn % 2 == 0)
            for name, eager in m.state().items():
                np.testing.assert_array_equal(after[name], eager, err_msg=f"turn {turn}: {name}")
    for r in graphs:
        r.close()


def test_a_recorded_call_without_its_own_scratch_is_refused(hip):
    m = Layer()
    assert K.sdpa_prefix_scratch(m.sdpa_args) > 0
    m.sdpa_args.scratch, m.sdpa_args.scratch_bytes = None, 0
    r = Recorded(lambda s: hip.sdpa_prefix(m.sdpa_args, s))
    assert r.error and "needs its own scratch" in r.error
    r.close()
    m.prefill(hip)  # and the backend goes on working
    m.calls(hip, scratch=False)


def test_backends_in_threads(hip):
    """One backend a thread, each with its own layer: every thread's results are those of a run by itself."""
    def run(be, seed):
        m = Layer(seed=seed)
        m.prefill(be)
        for _ in range(5):
            n = m.place()
            put(m.qkv, narrow(m.rng.standard_normal((m.nb, m.row)), DT))
            before = m.state()
            m.calls(be, scratch=False)
            m.check(before, m.state(), n)
        return m.state()

    alone = [run(hip, s) for s in range(3)]
    got, errors = [None] * 3, []

    def worker(i):
        try:
            got[i] = run(K.HipBackend(), i)
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            errors.append(f"thread {i}: {e!r}")

    threads = [threading.Thread(target=worker, args=(i,), daemon=True) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for a, b in zip(alone, got):
        for name in a:
            np.testing.assert_array_equal(a[name], b[name], err_msg=name)
