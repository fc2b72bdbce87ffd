"""Calls of the sampler of different sizes beside one another: captured, from several threads, through the C entry."""
import ctypes as C
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


class Desc(C.Structure):
    _fields_ = ([(n, C.c_longlong) for n in ("type", "R", "V")] + [("logits", C.c_void_p), ("ld", C.c_longlong), ("uniform", C.c_void_p)] +
                [(n, C.c_void_p) for n in ("temp_rows", "p_rows", "min_rows", "k_rows")] + [(n, C.c_double) for n in ("temp", "p", "min_p")] +
                [("k", C.c_longlong), ("token", C.c_void_p), ("logprob", C.c_void_p), ("cluster", C.c_longlong)])


def _rows(seed, R, V):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return 2.0 * torch.randn(R, V, generator=g, device="cuda"), torch.rand(R, generator=g, device="cuda")


def test_a_small_vocabulary_between_a_large_ones_capture_and_replay(cuda_device):
    from frankentorch_b200.ops import decode as D
    big, small = _rows(1, 2, 300000), _rows(2, 2, 700)
    kw = dict(top_p=0.9)
    want = [D.sample(*big, **kw), D.sample(*small, **kw)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [D.sample(*big, **kw), D.sample(*small, **kw), D.sample(*big, **kw)]
    for _ in range(3):
        again = D.sample(*small, **kw)
        graph.replay()
        for a, b in zip(got + [again], [want[0], want[1], want[0], want[1]]):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_threads_of_different_vocabularies(cuda_device):
    from frankentorch_b200.ops import decode as D
    sizes = (700, 300000, 40000)
    rows = [_rows(i, 2, V) for i, V in enumerate(sizes)]
    want = [D.sample(*x, top_k=20) for x in rows]
    got, errors = [None] * 3, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i] = D.sample(*rows[i], top_k=20)
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # shown by the test's thread
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_the_entry_takes_calls_of_threads_at_once(cuda_device):
    """Nothing that one call sets is in the way of another between its setting and its launch."""
    from frankentorch_b200.ops import _lib
    from frankentorch_b200.ops import decode as D
    entry = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p)(C.cast(_lib.load().ftk_sample, C.c_void_p).value)      # lets other threads run
    sizes = (9000, 300000)
    rows = [_rows(i, 1, V) for i, V in enumerate(sizes)]
    want = [D.sample(*x) for x in rows]
    out = [(torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")) for _ in sizes]
    streams = [torch.cuda.Stream() for _ in sizes]
    torch.cuda.synchronize()
    status = [set(), set()]

    def work(i):
        x, u = rows[i]
        d = Desc(type=2, R=1, V=sizes[i], logits=x.data_ptr(), ld=x.stride(0), uniform=u.data_ptr(),      # 2: fp32
                 temp=1.0, p=1.0, min_p=0.0, k=0, token=out[i][0].data_ptr(), logprob=out[i][1].data_ptr())
        for _ in range(2000):
            status[i].add(entry(C.byref(d), streams[i].cuda_stream))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [{0}, {0}]
    for a, b in zip(out, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
