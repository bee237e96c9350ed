"""The calls on device buffers on several streams."""
import ctypes as C

import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import dev
from hipmem import DevBuf, check, hip as hiprt, synchronize
from kurumi_amd import DType
from kutest import f32_to_bf16_bits
from test_gpu_linear_e4m3 import quantise_rows
from test_gpu_sdpa_prefix import Case

pytestmark = pytest.mark.gpu


def test_attention_beside_a_linear_on_another_stream(hip):
    """Each orders its own calls on one stream of its own: neither has the other's workspace. Every round
    starts both, and either's results are those of a run by itself."""
    streams = [C.c_void_p(), C.c_void_p()]
    for s in streams:
        check(hiprt().hipStreamCreate(C.byref(s)), "hipStreamCreate")
    m, n, k = 2048, 2048, 4096
    rng = np.random.default_rng(1)
    x = dev(f32_to_bf16_bits(rng.standard_normal((m, k), np.float32)))
    wq, sw = (dev(a) for a in quantise_rows(rng.standard_normal((n, k), np.float32)))
    y = DevBuf(2 * m * n)
    c = Case(DType.BF16, 20, 1, 16, 4, 128, 5000, 600, page=16)
    args = c.args()

    def linear(stream):
        hip.linear_e4m3(x.ptr, DType.BF16, wq.ptr, sw.ptr, y.ptr, DType.BF16, m, n, k, stream)

    def alone():
        hip.sdpa_prefix(args)
        synchronize()
        linear(None)
        return (*c.results(), y.numpy(np.uint16, (m, n)))

    want = alone()
    for turn in range(12):
        print(f"turn {turn}", flush=True)
        for _ in range(3):
            hip.sdpa_prefix(args, streams[0].value)
            linear(streams[1].value)
            hip.sdpa_prefix(args, streams[0].value)
        got = (*c.results(), y.numpy(np.uint16, (m, n)))
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a, b)
    for s in streams:
        check(hiprt().hipStreamDestroy(s), "hipStreamDestroy")


NULL_STREAM = 1  # hipStreamLegacy: the null stream, which a handle of 0 does not name in these calls


@pytest.mark.parametrize("call", ["rope", "sdpa_prefix", "logits_adjust"])
def test_the_null_stream_by_its_handle(hip, call):
    """A program whose work is on the null stream: long copies, then the inputs' true values, the call, and the copy of
    its outputs, with no wait between them. (With no handle the call is on the backend's own stream and would
    not wait.) Every round gives the results of a run that waits after each step."""
    L = hiprt()
    to_device = 3  # hipMemcpyDeviceToDevice
    L.hipMemcpyAsync.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int, C.c_void_p]
    rng = np.random.default_rng(2)
    rows, n = 64, 4096
    good, other = (dev(rng.standard_normal((rows, n)).astype(np.float32)) for _ in range(2))
    x, y, z = (DevBuf(4 * rows * n) for _ in range(3))
    long_a, long_b = DevBuf(1 << 30), DevBuf(1 << 30)
    d, heads = 64, n // 64
    keep = [dev(np.arange(rows, dtype=np.int32)), K.rope_freqs(d), dev(rng.standard_normal((300, d)).astype(np.float32))]
    if call == "rope":
        args = K.RopeArgs(dtype=DType.F32, scale=1.0, tokens=rows, q_heads=heads, head_dim=d, rot_dim=d, freqs=keep[1], positions=keep[0].ptr, q=x.ptr,
                          q_token_stride=n, q_head_stride=d, q_out=y.ptr, q_out_token_stride=n, q_out_head_stride=d)
    elif call == "sdpa_prefix":
        args = K.SdpaPrefixArgs(dtype=DType.F32, scale=0.125, batch=rows, q_len=1, q_heads=heads, kv_heads=1, head_dim=d, q=x.ptr, q_batch_stride=n,
                                q_token_stride=n, q_head_stride=d, out=y.ptr, out_batch_stride=n, out_token_stride=n, out_head_stride=d, prefix_len=300,
                                prefix_k=keep[2].ptr, prefix_v=keep[2].ptr, prefix_row_stride=d, prefix_head_stride=d)
    else:
        args = K.LogitsArgs(dtype=DType.F32, out_dtype=DType.F32, rows=rows, vocab=n, logits=x.ptr, logits_stride=n, out=y.ptr, out_stride=n)
    run = getattr(hip, call)

    def copy(dst, src, nbytes):
        check(L.hipMemcpyAsync(dst.ptr, src.ptr, nbytes, to_device, None), "hipMemcpyAsync")

    copy(x, good, 4 * rows * n)
    synchronize()
    run(args)
    want = y.numpy(np.float32, (rows, n))
    for _ in range(4):
        copy(x, other, 4 * rows * n)
        synchronize()
        copy(long_a, long_b, 1 << 30)
        copy(x, good, 4 * rows * n)
        run(args, NULL_STREAM)
        copy(z, y, 4 * rows * n)
        np.testing.assert_array_equal(z.numpy(np.float32, (rows, n)), want)


def small_calls(hip):
    """One small call of each kind, and what it writes."""
    c = Case(DType.F32, 2, 1, 4, 2, 64, 300, 20)
    args = c.args()
    rows, vocab, d = 3, 500, 64
    x, y = dev(np.ones((rows, vocab), np.float32)), dev(np.zeros((rows, vocab), np.float32))
    logits = K.LogitsArgs(dtype=DType.F32, out_dtype=DType.F32, rows=rows, vocab=vocab, logits=x.ptr, logits_stride=vocab, out=y.ptr, out_stride=vocab)
    q, qo, pos = dev(np.ones((rows, d), np.float32)), dev(np.zeros((rows, d), np.float32)), dev(np.zeros(rows, np.int32))
    rope = K.RopeArgs(dtype=DType.F32, scale=1.0, tokens=rows, q_heads=1, head_dim=d, rot_dim=d, freqs=K.rope_freqs(d), positions=pos.ptr, q=q.ptr,
                      q_token_stride=d, q_head_stride=d, q_out=qo.ptr, q_out_token_stride=d, q_out_head_stride=d)
    keep = (x, q, pos)
    return [(lambda: hip.rope(rope), lambda: qo.numpy(np.float32, (rows, d)), keep), (lambda: hip.sdpa_prefix(args), lambda: c.results()[0], keep),
            (lambda: hip.logits_adjust(logits), lambda: y.numpy(np.float32, (rows, vocab)), keep)]


def test_an_error_of_an_earlier_call_is_not_the_launchs(hip):
    """A call that the runtime refused (a device that is none) leaves its error with the thread: the launches that
    follow are none the worse, and the error is still there for the program to see."""
    L = hiprt()
    for call, result, _ in small_calls(hip):
        call()  # what is loaded at a first use is there
        want = result()
        L.hipGetLastError()
        assert L.hipSetDevice(1 << 20) != 0
        call()
        assert L.hipGetLastError() != 0
        np.testing.assert_array_equal(result(), want)
