"""What the copy of the hidden states that count refuses, before anything is launched (no GPU needed)."""
import ctypes
import os

import pytest


@pytest.fixture(scope="module")
def lib():
    from picotron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    return _lib.lib()


def test_rows_that_count(lib):
    def call(x=4096, t=4096, out=4096, rows=10, hidden=128, vocab=1000, ldx=128):
        P = ctypes.c_void_p
        return lib.pico_linear_log_probs_counted(P(x), P(t), P(out), rows, hidden, vocab, ldx, -100, None)
    for over in (dict(rows=-1), dict(hidden=0), dict(hidden=-8), dict(hidden=100), dict(vocab=0), dict(vocab=1 << 31), dict(rows=1 << 31, hidden=1 << 10), dict(rows=1 << 40),
                 dict(hidden=1 << 40, ldx=1 << 40)):
        assert call(**over) == -3, over
    for over in (dict(ldx=120), dict(ldx=132)):
        assert call(**over) == -5, over
    for over in (dict(x=None), dict(t=None), dict(out=None)):
        assert call(**over) == -1, over
    for over in (dict(x=4104), dict(t=4100), dict(out=4098)):
        assert call(**over) == -4, over
    assert call(rows=0, x=None, t=None, out=None) == 0
