"""Scratch memory of calls that run several launches (kernels.workspace), on the CPU."""
import threading

import pytest
import torch

from ml_music_style_transfer_amd import _lib as L
from ml_music_style_transfer_amd import kernels as K


@pytest.fixture
def one_stream(monkeypatch):
    monkeypatch.setattr(L, "stream", lambda: L.c_void_p(0))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def test_threads_on_one_stream_have_their_own(one_stream):
    """What a call's first launch leaves for its second must not be another thread's scratch: the
    threads' launches mix on the stream in any order."""
    dev, got, both = torch.device("cpu"), {}, threading.Barrier(2, timeout=30)

    def call(k):
        for n in (64, 4096, 64):  # 4096: outgrows the first
            both.wait()
            buf, size = K.workspace(n, dev)
            assert size == 4 * buf.numel() >= n
            got[k] = buf
            both.wait()
            if k == 0:
                assert got[0].data_ptr() != got[1].data_ptr()
            both.wait()
    errors = []

    def run(k):
        try:
            call(k)
        except BaseException as e:
            errors.append(e)
            both.abort()
    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_a_thread_keeps_its_buffer(one_stream):
    dev = torch.device("cpu")
    a, size = K.workspace(64, dev)
    assert K.workspace(size, dev)[0] is a
    assert K.workspace(0, dev) == (None, 0)
