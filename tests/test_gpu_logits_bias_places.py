"""ku_hip_logits_adjust with bias lists whose places are counted up to 2^31 - 1."""
import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import dev
from hipmem import DevBuf, check, hip as hiprt, synchronize
from kurumi_amd import DType

pytestmark = pytest.mark.gpu


def test_lists_at_the_end_of_the_longest_array(hip):
    """Rows whose entries lie in the last 700 places of 2^31 - 1 (8 GiB of ids, 8 GiB of values): a work-group's places
    run on past the last one. One list ends in the last 512 places, one starts there, one is the last place."""
    n, vocab = 2 ** 31 - 1, 900
    ids, values = DevBuf(4 * n), DevBuf(4 * n)
    rng = np.random.default_rng(3)
    tail = 700
    tail_ids, tail_values = rng.permutation(vocab)[:tail].astype(np.int32), rng.standard_normal(tail).astype(np.float32)
    for buf, part in ((ids, tail_ids), (values, tail_values)):
        check(hiprt().hipMemcpy(buf.ptr + 4 * (n - tail), part.ctypes.data, part.nbytes, 1), "hipMemcpy H2D")
    cuts = np.array([0, 400, 699, 700])
    offsets = dev((n - tail + cuts).astype(np.int32))
    for repeats in (False, True):
        if repeats:  # a list that names an id twice is added by another loop
            tail_ids[[1, 401]] = tail_ids[[0, 400]]
            check(hiprt().hipMemcpy(ids.ptr + 4 * (n - tail), tail_ids.ctypes.data, tail_ids.nbytes, 1), "hipMemcpy H2D")
        x, y = dev(np.zeros((3, vocab), np.float32)), DevBuf(12 * vocab)
        hip.logits_adjust(K.LogitsArgs(dtype=DType.F32, out_dtype=DType.F32, rows=3, vocab=vocab, logits=x.ptr, logits_stride=vocab, out=y.ptr,
                                       out_stride=vocab, bias_ids=ids.ptr, bias_values=values.ptr, bias_offsets=offsets.ptr, bias_count=n))
        synchronize()
        want = np.zeros((3, vocab), np.float32)
        for r in range(3):
            for i in range(cuts[r], cuts[r + 1]):
                want[r, tail_ids[i]] += tail_values[i]
        np.testing.assert_array_equal(y.numpy(np.float32, (3, vocab)), want)
