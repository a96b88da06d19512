"""The learner's operators without a GPU: what they refuse, and the sizes they ask for."""

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from mymyr_b200 import _lib, learn  # noqa: E402


def test_tensors_of_the_host_are_refused():
    x, y = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: learn.logprobs(x, y), lambda: learn.embedding(y, x), lambda: learn.adamw_state([x]),
                lambda: learn.adamw_step([x], [x], x, x, step=1), lambda: learn.AdamW([x])):
        with pytest.raises(ValueError):
            bad()


def test_embedding_workspace_grows_with_the_tokens():
    a = _lib.EmbeddingArgs()
    a.token_bits, a.vocabulary, a.width = 64, 1000, 16
    sizes = []
    for n in (0, 1, 5000, 10 ** 6):
        a.count = n
        sizes.append(_lib.lib().b2_embedding_workspace(C.byref(a)))
    assert sizes == sorted(sizes) and sizes[-1] >= 16 * 10 ** 6  # keys and places, twice
    assert _lib.lib().b2_embedding_workspace(None) == 0


def test_null_contexts_are_refused():
    L = _lib.lib()
    assert L.b2_logprobs(None, C.byref(_lib.LogprobsArgs()), None) == _lib.B2_INVALID_ARGUMENT
    assert L.b2_embedding(None, C.byref(_lib.EmbeddingArgs()), None, 0, None, None) == _lib.B2_INVALID_ARGUMENT
    assert L.b2_adamw(None, C.byref(_lib.AdamwArgs()), None) == _lib.B2_INVALID_ARGUMENT
    assert "null" in _lib.last_error()
