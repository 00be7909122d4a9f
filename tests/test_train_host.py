"""CPU tests of the table-training operators: the C ABI's refusals (checked
before any device call) and the Python entry points' argument errors."""
import ctypes as C

import pytest


def _call(name, *args):
    from ai_b200 import _lib

    return getattr(_lib.lib(), name)(*args)


P = C.c_void_p(4096)  # an address no refused call reads


@pytest.mark.parametrize("args", [
    (P, 7, 10, 4, 4, P, 3, 1.0, -1, P, 0, 4, None),       # table type
    (P, 0, 10, 4, 4, P, 3, 1.0, -1, P, 3, 4, None),       # output type
    (P, 0, 10, 4, 3, P, 3, 1.0, -1, P, 0, 4, None),       # table stride
    (P, 0, 10, 4, 4, P, 3, 1.0, -1, P, 0, 3, None),       # output stride
    (P, 0, 10, 0, 4, P, 3, 1.0, -1, P, 0, 4, None),       # no columns
    (P, 0, 10, 4, 4, P, -1, 1.0, -1, P, 0, 4, None),      # negative tokens
    (P, 0, 1 << 31, 4, 4, P, 3, 1.0, -1, P, 0, 4, None),  # vocabulary past int32
    (None, 0, 10, 4, 4, P, 3, 1.0, -1, P, 0, 4, None),    # null table
    (P, 0, 10, 4, 4, None, 3, 1.0, -1, P, 0, 4, None),    # null ids
])
def test_embedding_refusals(args):
    from ai_b200 import _lib

    assert _call("fg_embedding", *args) == _lib.FG_EINVAL
    assert b"fg_embedding" in _lib.lib().fg_last_error()


def test_embedding_of_no_tokens_needs_no_device():
    assert _call("fg_embedding", P, 0, 10, 4, 4, None, 0, 1.0, -1, None, 0, 4, None) == 0


@pytest.mark.parametrize("args", [
    (P, 9, 4, P, 3, 10, 4, 1.0, -1, P, 0, 4, 0, None),
    (P, 0, 4, P, 3, 10, 4, 1.0, -1, P, 9, 4, 0, None),
    (P, 0, 3, P, 3, 10, 4, 1.0, -1, P, 0, 4, 0, None),
    (P, 0, 4, P, 3, 10, 4, 1.0, -1, P, 0, 3, 0, None),
    (P, 0, 4, P, 3, -1, 4, 1.0, -1, P, 0, 4, 0, None),
    (None, 0, 4, P, 3, 10, 4, 1.0, -1, P, 0, 4, 0, None),
    (P, 0, 4, P, 3, 10, 4, 1.0, -1, None, 0, 4, 0, None),
])
def test_embedding_grad_refusals(args):
    from ai_b200 import _lib

    assert _call("fg_embedding_grad", *args) == _lib.FG_EINVAL
    assert b"fg_embedding_grad" in _lib.lib().fg_last_error()


@pytest.mark.parametrize("args", [
    (P, 0, 4, P, 3, 10, 4, 1.0, -1, None, P, 0, 4, P, None),
    (P, 0, 4, P, 3, 10, 4, 1.0, -1, P, P, 0, 4, None, None),
    (P, 0, 4, P, 3, 10, 4, 1.0, -1, P, None, 0, 4, P, None),
    (P, 0, 4, P, 3, 10, 0, 1.0, -1, P, P, 0, 4, P, None),
])
def test_embedding_grad_rows_refusals(args):
    from ai_b200 import _lib

    assert _call("fg_embedding_grad_rows", *args) == _lib.FG_EINVAL


@pytest.mark.parametrize("args", [
    (P, 5, 2, 8, 8, P, 1.0, 0, P, P, P, None, None, None),             # type
    (P, 0, 2, 0, 8, P, 1.0, 0, P, P, P, None, None, None),             # no columns
    (P, 0, 2, 8, 7, P, 1.0, 0, P, P, P, None, None, None),             # stride
    (P, 0, 2, 8, 8, P, 0.0, 0, P, P, P, None, None, None),             # scale
    (P, 0, 2, 8, 8, P, float("inf"), 0, P, P, P, None, None, None),
    (P, 0, 2, 8, 8, P, float("nan"), 0, P, P, P, None, None, None),
    (P, 0, 2, 8, 8, P, 1.0, 9, P, P, P, P, P, None),                   # more alternatives than columns
    (P, 0, 2, 80, 80, P, 1.0, 65, P, P, P, P, P, None),                # more than FG_MAX_TOP
    (P, 0, 2, 8, 8, P, 1.0, 2, P, P, P, None, P, None),                # null
    (P, 0, 2, 8, 8, None, 1.0, 0, P, P, P, None, None, None),
])
def test_log_probs_refusals(args):
    from ai_b200 import _lib

    assert _call("fg_log_probs", *args) == _lib.FG_EINVAL
    assert b"fg_log_probs" in _lib.lib().fg_last_error()


@pytest.mark.parametrize("args", [
    (P, 5, 2, 8, 8, P, 1.0, P, P, P, None, P, 8, None),
    (P, 0, 2, 8, 8, P, 1.0, P, P, P, None, P, 7, None),
    (P, 0, 2, 8, 8, P, -1.0, P, P, P, None, P, 8, None),
    (P, 0, 2, 8, 8, P, 1.0, P, None, P, P, P, 8, None),  # dentropy without entropy
    (P, 0, 2, 8, 8, P, 1.0, None, P, P, None, P, 8, None),
])
def test_log_probs_grad_refusals(args):
    from ai_b200 import _lib

    assert _call("fg_log_probs_grad", *args) == _lib.FG_EINVAL


def test_clip_refusals():
    from ai_b200 import _lib

    ptrs, sizes, types = (C.c_void_p * 1)(4096), (C.c_int64 * 1)(8), (C.c_int * 1)(0)
    ok = (1, ptrs, sizes, types, None)
    for bad in ((*ok, -1.0, P, None), (*ok, float("nan"), P, None), (*ok, 1.0, None, None),
                (-1, ptrs, sizes, types, None, 1.0, P, None),
                (1, None, sizes, types, None, 1.0, P, None),
                (1, ptrs, (C.c_int64 * 1)(-1), types, None, 1.0, P, None),
                (1, ptrs, sizes, (C.c_int * 1)(4), None, 1.0, P, None),
                (1, (C.c_void_p * 1)(None), sizes, types, None, 1.0, P, None),
                (1, ptrs, sizes, types, (C.c_void_p * 1)(None), 1.0, P, None)):
        assert _call("fg_clip_grad_norm", *bad) == _lib.FG_EINVAL
        assert b"fg_clip_grad_norm" in _lib.lib().fg_last_error()


def test_python_refuses_host_tensors():
    import torch

    from ai_b200 import train

    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: train.Embedding(x, i), lambda: train.EmbeddingGrad(x, i, 10),
                 lambda: train.EmbeddingGradRows(x, i, 10), lambda: train.LogProbs(x, i),
                 lambda: train.LogProbsGrad(x, i, x[:, 0], x[:, 0]), lambda: train.ClipGradNorm([x], 1.0),
                 lambda: train.ClipGradNorm([], 1.0), lambda: train.ClipGradNorm([x], -1.0)):
        with pytest.raises(train.TensorError):
            call()


def test_log_probs_peak_refusals():
    from ai_b200 import _lib

    for args in ((P, 0, 2, 8, 7, P, 1.0, 0, P, P, P, P, None, None, None),   # stride
                 (P, 0, 2, 8, 8, P, 1.0, 9, P, P, P, P, P, P, None),         # more alternatives than columns
                 (P, 0, 2, 8, 8, P, 1.0, 0, P, P, None, P, None, None, None)):  # null
        assert _call("fg_log_probs_peak", *args) == _lib.FG_EINVAL
    for args in ((P, 0, 2, 8, 8, P, 1.0, None, P, P, None, P, 8, None),      # no peak
                 (P, 0, 2, 8, 8, P, 1.0, P, None, P, P, P, 8, None),         # dentropy without entropy
                 (P, 0, 2, 8, 8, P, 0.0, P, P, P, None, P, 8, None)):
        assert _call("fg_log_probs_grad_peak", *args) == _lib.FG_EINVAL


@pytest.mark.parametrize("current,device,want", [(0, None, 0), (1, None, 1), (1, "cuda", 1), (0, "cuda:1", 1), (1, "cuda:0", 0), (0, 2, 2)])
def test_check_waits_for_the_device_asked_for_and_goes_back(monkeypatch, current, device, want):
    """"cuda" is the current device, and the caller's current device is the
    same afterwards although fg_synchronize makes its own current; also where
    it reports an id."""
    import torch

    from ai_b200 import _lib, train

    state = {"current": current, "asked": [], "rc": 0}

    class Library:
        @staticmethod
        def fg_synchronize(index):
            state["asked"].append(index)
            state["current"] = index
            return state["rc"]

        @staticmethod
        def fg_last_error():
            return b"an id"

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["current"] = state["current"], self.index

        def __exit__(self, *exc):
            state["current"] = self.before

    monkeypatch.setattr(_lib, "lib", lambda: Library)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    train.Check(device)
    assert state["asked"] == [want] and state["current"] == current
    state["rc"] = _lib.FG_EINVAL
    with pytest.raises(_lib.FGError):
        train.Check(device)
    assert state["asked"] == [want] * 2 and state["current"] == current


def test_check_refuses_a_host_device():
    from ai_b200 import train

    with pytest.raises(train.TensorError):
        train.Check("cpu")
