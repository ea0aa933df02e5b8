"""The recurrence over a long axis of few rows, whose rows are cut into segments that pass their maps through
a workspace (gated.hip), and over more than 2^31 elements."""
import threading

import pytest
import torch

from ml_music_style_transfer_amd import _lib as L
from ml_music_style_transfer_amd import engine as E
from ml_music_style_transfer_amd import train as T
from oracle import gated_ref as R
from test_gated import IDS, TYPES, _check, _data, _run, _within


def _segmented(B, C, T, dtype):
    return L.load().mst_gated_workspace_size(L.TYPES[dtype], B, C, T) > 0


def test_these_rows_are_cut():
    for dtype in TYPES:
        assert _segmented(1, 3, 10741, dtype) and _segmented(1, 16, 12001, dtype) and _segmented(2, 3, 10741, dtype)
        assert not _segmented(1, 16, 6000, dtype) and not _segmented(27000, 4, 20011, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("padded", [False, True], ids=["full", "padded"])
@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_every_type_and_direction(cuda, dtype, reverse, padded):
    T_ = 10741
    x, gate, gh, h0, gl = _data(2, 3, T_, dtype, seed=3, shift=3.0)
    n = torch.tensor([T_ - 601, T_ // 3], dtype=torch.int32) if padded else None
    _check(cuda, x, gate, gh, h0, gl, n, reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
def test_captured_twice(cuda, reverse):
    """Two graphs of the forward and backward, replayed in turn with eager calls between: each holds a
    workspace of its own."""
    static = [t.to(cuda) for t in _data(1, 16, 12001, seed=4)]

    def program():
        a, b, c = (t.detach().requires_grad_() for t in (static[0], static[1], static[3]))
        h, last = E.gated_recurrence(a, b, c, None, reverse)
        return (h, last, *torch.autograd.grad((h, last), (a, b, c), (static[2], static[4])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        program()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, program()))
    for k in range(3):
        for s, t in zip(static, _data(1, 16, 12001, seed=30 + k)):
            s.copy_(t)
        for graph, _ in graphs:
            graph.replay()
        want = program()
        torch.cuda.synchronize()
        for _, out in graphs:
            for u, v in zip(out, want):
                assert torch.equal(u, v)


@pytest.mark.gpu
def test_streams_at_once(cuda):
    cases = [_data(1, 16, 12001, seed=40 + k) for k in range(3)]
    want = [_run(cuda, *case[:3], h0=case[3], gl=case[4]) for case in cases]
    dev = [[t.to(cuda) for t in case] for case in cases]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in cases]
    for s, d in zip(streams, dev):
        with torch.cuda.stream(s):
            got.append(_run(cuda, *d[:3], h0=d[3], gl=d[4]))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for u, v in zip((a[0], a[1], *a[2]), (b[0], b[1], *b[2])):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_threads_on_one_stream(cuda):
    """Host threads whose launches mix on the default stream: each call's maps and partial sums are its own."""
    cases = [[t.to(cuda) for t in _data(1, 16, 12001, seed=50 + k)] for k in range(3)]

    def call(case):
        x, gate, gh, h0, gl = case
        h, last, grads = _run(cuda, x, gate, gh, h0, gl)
        p = torch.empty_like(x).requires_grad_()
        p.grad = x
        return (h, last, *grads, T.grad_norm([p]))
    want = [call(case) for case in cases]
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(len(cases), timeout=60)

    def run(k):
        try:
            start.wait()
            got = [call(cases[k]) for _ in range(20)]
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for out in got for u, v in zip(out, want[k]))
        except BaseException as e:
            failed.append((k, e))
    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.gpu
def test_more_than_2_to_the_31_elements(cuda):
    """Every row is the same expanded one: all rows equal, and that row within the oracle's bounds over its
    whole length, forward and backward."""
    B, C, T_ = 27000, 4, 20011
    assert B * C * T_ > 2 ** 31
    x, gate, gh, h0, gl = _data(1, 1, T_, torch.bfloat16, seed=9)
    leaves = [t.to(cuda).expand(B, C, *t.shape[2:]).detach().requires_grad_() for t in (x, gate, h0)]
    h, last = E.gated_recurrence(*leaves)
    f = R.forward(x, gate, h0)
    b = R.backward(f, gh, gl)

    def same(t, ref, err, what):
        assert (t == t[:1, :1]).all(), what
        _within(t[:1, :1], ref, err, what)
    same(h, f["h"], f["h_err"], "h")
    same(last, f["last"], f["last_err"], "last")
    dev = [t.to(cuda).expand(B, C, *t.shape[2:]) for t in (gh, gl)]
    grads = torch.autograd.grad((h, last), leaves, dev)
    del h
    for t, k in zip(grads, ("dx", "dgate", "dh0")):
        same(t, b[k], b[k + "_err"], k)
