"""What the copy of the hidden states that count refuses, and forward-mode tangents, before anything is launched (no GPU needed)."""
import ctypes
import os

import pytest
import torch


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


def forward_mode(device):
    from torch.autograd import forward_ad

    from picotron_amd.functional import linear_log_probs, log_probs, policy_loss, preference_loss
    t = torch.zeros(2, 3, dtype=torch.long, device=device)
    A = torch.zeros(2, 1, device=device)
    with forward_ad.dual_level():
        for grad in (False, True):
            x, w = torch.zeros(2, 3, 128, dtype=torch.bfloat16, device=device), torch.zeros(40, 128, dtype=torch.bfloat16, device=device)
            dual, wdual = (forward_ad.make_dual(v.requires_grad_(grad), torch.ones_like(v)) for v in (x, w))
            for call in (lambda: log_probs(dual, t), lambda: log_probs(dual, t, entropy=True), lambda: policy_loss(dual, t, A), lambda: preference_loss(dual, t),
                         lambda: linear_log_probs(dual, w, t), lambda: linear_log_probs(x, wdual, t)):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()


def test_forward_mode_tangents():
    """They would be lost without a sign."""
    forward_mode("cpu")


@pytest.mark.gpu
def test_forward_mode_tangents_on_the_gpu(device):
    forward_mode(device)
