"""Rows of class scores from several threads of the host at once, through the C-ABI (which gives
up Python's lock during a call)."""
import ctypes
import threading

import pytest
import torch

from k2_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
CALLS = 1500


def rows_of(x):
    return _lib.ClassRows(scores=x.data_ptr(), type=0, num_classes=x.shape[1], outer=1,
                          inner=x.shape[0], outer_stride=0, inner_stride=x.shape[1])


def token_calls(x):
    """Top classes: a block's shared memory holds a row."""
    n = x.shape[0]
    values = torch.zeros(n, 4, device=DEV)
    classes = torch.zeros(n, 4, dtype=torch.int32, device=DEV)
    r, stream = rows_of(x), torch.cuda.Stream()

    def call():
        return _lib.lib.k2b200_token_scores(
            ctypes.byref(r), None, 0, 4, None, None, values.data_ptr(), classes.data_ptr(), None,
            stream.cuda_stream)
    return call, lambda: torch.equal(classes.long(), torch.topk(x, 4).indices)


def distil_calls(x):
    n, c = x.shape
    r, stream = rows_of(x), torch.cuda.Stream()
    tokens = torch.arange(n, device=DEV, dtype=torch.int32)
    of_teacher, loss = torch.zeros(n, device=DEV), torch.full((n,), -1.0, device=DEV)
    t = _lib.Teacher(tokens=tokens.data_ptr(), tokens_64=0, scores=of_teacher.data_ptr(), type=0,
                     entries=1, temperature=1.0, weight=1.0, reduction=0)

    def call(keep=(x, tokens, of_teacher)):
        return _lib.lib.k2b200_distillation(
            ctypes.byref(r), ctypes.byref(t), loss.data_ptr(), None, None, 0, 0, None, 0,
            stream.cuda_stream)
    want = -torch.log_softmax(x.double(), 1)[torch.arange(n), tokens.long()]
    # (sums of up to 49000 terms, a thread's 200 one after the other, and a logarithm)
    return call, lambda: bool(((loss - want).abs() <= 512 * 2.0 ** -24 * (want.abs() + 1)).all())


@pytest.mark.parametrize("make", [token_calls, distil_calls])
def test_threads_with_rows_of_unlike_lengths(make):
    """One kernel with 57 KB of shared memory in one thread and 190 in another: neither takes away
    what the other one asked for."""
    g = torch.Generator(device=DEV).manual_seed(0)
    work = [make(torch.randn(160, c, generator=g, device=DEV)) for c in (14500, 48000) * 2]
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(len(work))

    def run(call):
        start.wait()
        for _ in range(CALLS):
            if call() != 0:
                failed.append(_lib.lib.k2b200_last_error())
                return

    threads = [threading.Thread(target=run, args=(call,)) for call, _ in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    assert all(right() for _, right in work)
