"""A handle may be opened while a stream captures, on this thread or another: the capture holds, and so does the handle."""
import gc
import threading

import numpy as np
import pytest

from cache_reference import Case
from shim import q8_cache as C
from test_gpu_noalloc_streams import GLOBAL, THREAD_LOCAL, _Hip, _ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [GLOBAL, THREAD_LOCAL])
@pytest.mark.parametrize("thread", [False, True])
def test_opened_during_a_capture(mode, thread):
    rng = np.random.default_rng(1)
    case = Case(rng, [(1, 900), (1, 40)], 4, 2, 64, 16, longest=1)
    cache, batch = case.upload()
    q = C.Array.of(rng.normal(0, 1, (2, 256)), C.BF16)
    outs = [C.Array(2, 256, C.BF16) for _ in range(3)]
    hip = _Hip()
    stream = hip.stream()
    opened = []
    with C.Ops() as a:
        a.reserve(C.attention_workspace(C.BF16, cache, batch, 4))
        a.attention(C.BF16, cache, batch, 4, q, outs[0])
        a.synchronize()
        a.set_stream(stream.value)
        gc.collect()        # a buffer that an earlier test left in a cycle, freed during a capture, would end it
        gc.disable()
        hip.begin(stream, mode)
        try:
            a.attention(C.BF16, cache, batch, 4, q, outs[1])
            if thread:
                t = threading.Thread(target=lambda: opened.append(C.Ops()))
                t.start()
                t.join()
            else:
                opened.append(C.Ops())
        finally:
            exe = hip.end(stream)
            gc.enable()
        assert len(opened) == 1
        with opened[0] as b:
            b.attention(C.BF16, cache, batch, 4, q, outs[2])
            b.synchronize()
            _ok(hip.lib.hipGraphLaunch(exe, stream))
            a.synchronize()
        want = outs[0].numpy()
        assert np.any(want != 0) and all(np.array_equal(o.numpy(), want) for o in outs[1:])
        _ok(hip.lib.hipGraphExecDestroy(exe))
        a.set_stream(None)
    hip.lib.hipStreamDestroy(stream)
