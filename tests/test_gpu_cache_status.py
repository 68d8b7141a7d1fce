"""lfm_attention_status beside kernels of other streams, other threads and captures."""

import ctypes
import threading
import time

import pytest

from cache_attn_ref import ptr
from test_gpu_cache_attn import check, shape_of, status_of

pytestmark = pytest.mark.gpu

BAD_SLOT, BAD_LEN = 2, 4


class Call:
    """A decode of one session whose slot or length is out of range: a row of zeros and a report."""

    def __init__(self, slot, length):
        import torch
        self.sh = shape_of("f16", 1, 1, 64, 32)
        self.q, self.out = (torch.zeros(64, dtype=torch.float16, device="cuda") for _ in range(2))
        self.cache = torch.zeros(32 * 64, dtype=torch.float16, device="cuda")
        self.slots, self.lens = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (slot, length))

    def __call__(self, lib, stream):
        check(lib.lfm_attention_decode(self.sh, ptr(self.q), 64, ptr(self.cache), ptr(self.cache), 2048, 1,
                                       ptr(self.slots), ptr(self.lens), 1, 32, 0, 0, None, ptr(self.out), 64,
                                       ctypes.c_void_p(stream.cuda_stream)), "decode")


def status_on(lib, stream):
    s = ctypes.c_uint32(99)
    check(lib.lfm_attention_status(ctypes.byref(s), ctypes.c_void_p(stream.cuda_stream)), "status")
    return s.value


def test_no_report_of_another_stream_is_lost(cuda_lib):
    import torch
    call = Call(5, 3)
    work, watch = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    status_of(cuda_lib)
    lost = 0
    for i in range(4000):
        with torch.cuda.stream(work):
            torch.cuda._sleep(i % 400 * 300)  # up to some 60 us: the report falls before, into and behind the status
        call(cuda_lib, work)
        seen = status_on(cuda_lib, watch)
        work.synchronize()
        lost += (seen | status_on(cuda_lib, watch)) != BAD_SLOT
    assert lost == 0


def test_two_threads_take_every_report_between_them(cuda_lib):
    import torch
    calls = [Call(5, 3), Call(0, 40)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    status_of(cuda_lib)
    taken, lock, stop = [0], threading.Lock(), threading.Event()

    def watch(stream):
        torch.cuda.set_device(0)
        while not stop.is_set():
            got = status_on(cuda_lib, stream)
            with lock:
                taken[0] |= got

    threads = [threading.Thread(target=watch, args=(s,)) for s in streams[:2]]
    for t in threads:
        t.start()
    try:
        for _ in range(200):
            for c in calls:
                c(cuda_lib, streams[2])
            streams[2].synchronize()
            for _ in range(5000):
                with lock:
                    if taken[0] == BAD_SLOT | BAD_LEN:
                        break
                time.sleep(0.001)
            with lock:
                assert taken[0] == BAD_SLOT | BAD_LEN
                taken[0] = 0
    finally:
        stop.set()
        for t in threads:
            t.join()


def test_a_capture_refuses_the_status_and_goes_on(cuda_lib):
    import torch
    call = Call(5, 3)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    status_of(cuda_lib)
    s = ctypes.c_uint32(99)
    with torch.cuda.stream(side):
        graph.capture_begin(capture_error_mode="thread_local")
        call(cuda_lib, side)
        refused = cuda_lib.lfm_attention_status(ctypes.byref(s), ctypes.c_void_p(side.cuda_stream))
        message = cuda_lib.lfm_ops_error()
        call(cuda_lib, side)
        graph.capture_end()
    assert refused == 1 and b"captured" in message and s.value == 99
    torch.cuda.synchronize()
    assert status_of(cuda_lib) == 0
    graph.replay()
    torch.cuda.synchronize()
    assert status_of(cuda_lib) == BAD_SLOT
