"""What a commit reports when more than one thing went wrong in it: no condition hides another. A rank that never arrives is a
child process that only hands over its inbox; the wait for it is cut to 200 ms and returns."""
import os
import subprocess
import sys

import numpy as np
import pytest

from nuclis_b200 import Backend, KvCache, NuclisError, kv_spans
from test_gpu_wait_limit import CHILD, ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("span_first", [False, True])
def test_a_bad_span_does_not_hide_a_wait_that_ran_out(span_first):
    child = subprocess.Popen([sys.executable, "-c", CHILD], env=dict(os.environ, NU_ROOT=ROOT), stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True)
    b = Backend(0)
    try:
        theirs = bytes.fromhex(child.stdout.readline().strip())
        b.comm_attach_peers([b.comm_peer_handle(), theirs], rank=0)
        b.comm_set_wait_ms(200)
        shape = KvCache(1, 32, 1, 64)
        cache, spans, rows, total = b.create(shape.bytes), b.create(16), b.create(2 * 64 * 4), b.create(5120 * 4)
        spans.write(kv_spans([(0, 40, 1)]))
        total.write(np.ones(5120, dtype=np.float32))

        def read():
            b.kv_read(cache, shape, spans, 1, 1, rows.slice(0, 256), 64, rows.slice(256, 256), 64)
        b.begin()
        if span_first:
            read()
        b.allreduce_sum_f32(total, 5120)
        if not span_first:
            read()
        with pytest.raises(NuclisError) as e:
            b.commit()
        assert e.value.name == "ExecutionFailed" and "never arrived" in str(e.value) and "outside the key/value cache" in str(e.value)
        # each is told once
        spans.write(kv_spans([(0, 31, 1)]))
        b.begin()
        read()
        b.commit()
        b.comm_destroy()
    finally:
        child.stdin.write("done\n")
        child.stdin.flush()
        child.wait(timeout=60)
        b.deinit()
