"""What the operators on log-probabilities refuse, at the C ABI and in the host path, before anything is launched (no GPU needed)."""
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


def logits(data=4096, batch=2, seq=4, vocab=1000, dtype=0, **over):
    from picotron_amd._lib import Logits
    z = Logits(data, batch, seq, vocab, seq * vocab, vocab, dtype, 0)
    for k, v in over.items():
        setattr(z, k, v)
    return z


def tokens(data=4096):
    from picotron_amd._lib import PerRow
    return PerRow(data, 4, 1)


BUF = ctypes.c_void_p(4096)      # never read: every call here is refused first
R = ctypes.byref


def message(lib):
    return lib.pico_last_error().decode()


@pytest.mark.parametrize("over,code", [(dict(dtype=7), -2), (dict(vocab=0), -3), (dict(vocab=1 << 29), -3), (dict(batch=-1), -3), (dict(batch=1 << 20, seq=1 << 12), -3), (dict(batch=1 << 20, seq=5, vocab=40000), -3), (dict(batch=1 << 20, seq=40), -3),
                                       (dict(data=None), -1), (dict(data=4097), -4), (dict(row_stride=-8), -5), (dict(batch_stride=-8), -5)])
def test_logits_that_are_refused_everywhere(lib, over, code):
    from picotron_amd._lib import PerRow, Policy, PolicySaved
    z, t = logits(**over), tokens()
    v = PerRow(4096, 4, 1)
    p = Policy(v, v, v, v, 0.2, 0.2, 0.0, 0.0, 1.0)
    saved = PolicySaved(4096, 4096, 4096, 4096)
    assert lib.pico_log_probs_fwd(R(z), R(t), BUF, None, None, 1.0, -100, None) == code, message(lib)
    assert lib.pico_log_probs_bwd(R(z), R(t), BUF, None, R(v), None, None, 0, BUF, 4000, 1000, 1.0, -100, None) == code, message(lib)
    assert lib.pico_policy_loss_fwd(R(z), R(t), R(p), BUF, BUF, BUF, BUF, R(saved), None, 0, 0, 1.0, -100, None) == code, message(lib)
    assert lib.pico_preference_loss_fwd(R(z), R(t), None, 0.1, 0.0, 0, 1.0, BUF, BUF, BUF, BUF, None, BUF, -100, None) == code, message(lib)


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), float("inf"), 1e-38])
def test_temperatures(lib, temperature):
    assert lib.pico_log_probs_fwd(R(logits()), R(tokens()), BUF, None, None, temperature, -100, None) == -3
    assert "temperature" in message(lib)


def test_missing_pointers(lib):
    from picotron_amd._lib import PerRow, Policy, PolicySaved
    z, t, v, none = logits(), tokens(), PerRow(4096, 4, 1), PerRow(None, 0, 0)
    assert lib.pico_log_probs_fwd(None, R(t), BUF, None, None, 1.0, -100, None) == -1
    assert lib.pico_log_probs_fwd(R(z), None, BUF, None, None, 1.0, -100, None) == -1
    assert lib.pico_log_probs_fwd(R(z), R(tokens(None)), BUF, None, None, 1.0, -100, None) == -1
    assert lib.pico_log_probs_fwd(R(z), R(t), None, None, None, 1.0, -100, None) == -1
    assert lib.pico_log_probs_bwd(R(z), R(t), None, None, R(v), None, None, 0, BUF, 4000, 1000, 1.0, -100, None) == -1
    assert lib.pico_log_probs_bwd(R(z), R(t), BUF, None, R(none), R(none), None, 0, BUF, 4000, 1000, 1.0, -100, None) == -1
    assert lib.pico_log_probs_bwd(R(z), R(t), BUF, None, R(v), R(v), None, 0, BUF, 4000, 1000, 1.0, -100, None) == -1      # dentropy without entropy
    assert lib.pico_log_probs_bwd(R(z), R(t), BUF, None, R(v), None, None, 1, BUF, 4000, 1000, 1.0, -100, None) == -1      # have_unit without grad_out
    assert lib.pico_log_probs_bwd(R(z), R(t), BUF, None, R(v), None, None, 0, None, 4000, 1000, 1.0, -100, None) == -1
    saved, p = PolicySaved(4096, 4096, None, None), Policy(v, none, none, none, 0.2, 0.2, 0.0, 0.0, 1.0)

    def policy(p=p, saved=saved, d=None, loss=BUF):
        return lib.pico_policy_loss_fwd(R(z), R(t), R(p) if p else None, loss, BUF, BUF, BUF, R(saved) if saved else None, d, 4000, 1000, 1.0, -100, None)
    assert policy(p=None) == -1 and policy(loss=None) == -1
    assert policy(p=Policy(none, none, none, none, 0.2, 0.2, 0.0, 0.0, 1.0)) == -1
    assert policy(p=Policy(v, none, none, none, 0.2, 0.2, 0.1, 0.0, 1.0)) == -1 and "ref_log_probs" in message(lib)
    assert policy(saved=None, d=BUF) == -1 and policy(saved=PolicySaved(), d=BUF) == -1
    assert policy(p=Policy(v, none, none, none, 0.2, 0.2, 0.0, 0.5, 1.0), d=BUF) == -1                                     # entropy, nothing to keep it in
    assert policy(p=Policy(v, none, none, none, -0.1, 0.2, 0.0, 0.0, 1.0)) == -3 and "clip" in message(lib)
    assert policy(p=Policy(v, none, none, none, 0.2, float("nan"), 0.0, 0.0, 1.0)) == -3
    assert lib.pico_preference_loss_fwd(R(z), R(t), None, 0.1, 0.0, 0, 1.0, None, BUF, BUF, BUF, None, BUF, -100, None) == -1
    assert lib.pico_preference_loss_fwd(R(z), R(t), None, 0.1, 0.0, 0, 1.0, BUF, BUF, BUF, BUF, None, None, -100, None) == -1
    assert lib.pico_preference_loss_fwd(R(z), R(t), None, 0.1, 1.5, 0, 1.0, BUF, BUF, BUF, BUF, None, BUF, -100, None) == -3
    assert lib.pico_preference_loss_fwd(R(logits(batch=3)), R(t), None, 0.1, 0.0, 0, 1.0, BUF, BUF, BUF, BUF, None, BUF, -100, None) == -3 and "even" in message(lib)
    assert lib.pico_preference_loss_fwd(R(z), R(t), None, 0.1, 0.0, 0, 1.0, BUF, BUF, BUF, BUF, None, ctypes.c_void_p(4100), -100, None) == -4


@pytest.mark.parametrize("dtype,size", [(0, 2), (1, 4)])
def test_gradients_that_overlap_or_lie_otherwise(lib, dtype, size):
    from picotron_amd._lib import PerRow
    z, t, v = logits(dtype=dtype), tokens(), PerRow(4096, 4, 1)

    def bwd(d=4096, batch=4000, row=1000):
        return lib.pico_log_probs_bwd(R(z), R(t), BUF, None, R(v), None, None, 0, ctypes.c_void_p(d), batch, row, 1.0, -100, None)
    assert bwd(row=999) == -5 and bwd(batch=3999) == -5 and "overlap" in message(lib)
    assert bwd(d=4096 + size) == -4 and bwd(row=1001, batch=4008) == -4 and bwd(batch=4001) == -4


def test_linear_log_probs(lib):
    """Sizes, pitches, alignments, pointers and workspaces."""
    # x, partial results of three groups of 48 columns, three numbers a row and one more, each from a 16-byte boundary
    assert lib.pico_linear_log_probs_workspace_bytes(100, 72, 129) == 100 * 72 * 2 + 128 * 3 * 8 + 100 * 8 + 100 * 4 + 100 * 4 + 16
    for sizes in ((-1, 8, 8), (1, -8, 8), (1, 8, 1 << 40), (1 << 40, 8, 8)):
        assert lib.pico_linear_log_probs_workspace_bytes(*sizes) == -1

    def fwd(x=4096, w=4096, t=4096, lp=4096, ms=4096, M=10, K=128, N=1000, ldx=128, ldw=128, T=1.0, ws=4096, bytes=1 << 20):
        P = ctypes.c_void_p
        return lib.pico_linear_log_probs_fwd(P(x), P(w), P(t), P(lp), P(ms), M, K, N, ldx, ldw, T, -100, P(ws), bytes, None)

    def bwd(x=4096, w=4096, t=4096, ms=4096, g=4096, d=4096, M=10, K=128, N=1000, ldx=128, ldw=128, ldd=1000, T=1.0, ws=4096, bytes=1 << 20):
        P = ctypes.c_void_p
        return lib.pico_linear_log_probs_dlogits(P(x), P(w), P(t), P(ms), P(g), P(d), M, K, N, ldx, ldw, ldd, T, -100, P(ws), bytes, None)
    for call in (fwd, bwd):
        for over in (dict(M=-1), dict(K=64), dict(K=100), dict(N=0), dict(ldx=120), dict(ldw=132), dict(ldx=1 << 31), dict(K=0), dict(M=1 << 31), dict(T=0.0), dict(T=float("nan"))):
            assert call(**over) == -3, over
        for over in (dict(x=4104), dict(w=4098), dict(t=4100), dict(ms=4100), dict(ws=4100)):
            assert call(**over) == -4, over
        for over in (dict(x=None), dict(w=None), dict(t=None), dict(ws=None)):
            assert call(**over) == -1, over
        assert call(bytes=100) == -6 and "workspace" in message(lib)
    assert fwd(lp=None) == -1 and bwd(ms=None) == -1 and bwd(g=None) == -1 and bwd(d=None) == -1 and bwd(d=4104) == -4
    for ldd in (992, 1004, 1008):
        assert bwd(ldd=ldd) == -5 and "row pitch" in message(lib)
    assert bwd(N=1001, ldd=1001) == -5


def test_linear_log_probs_backward_of_the_rows_that_count(lib):
    """Sizes that it takes (workspaces in bytes) and does not (0), and what the call refuses."""
    size = lib.pico_linear_log_probs_bwd_workspace_bytes
    # d(logits), x, partial sums, four numbers a row, targets and positions, one number
    assert size(2000, 4096, 32000) == 2000 * 32000 * 2 + 2000 * 4096 * 2 + 2 ** 27 + 2000 * 16 + 2000 * 8 + 2000 * 4 + 16
    assert size(2000, 4096, 32001) == size(2000, 4096, 32008) > size(2000, 4096, 32000)
    assert size(2800, 576, 49152) > 0 and size(9000, 4096, 32000) > 9000 * (32000 * 2 + 4096 * 6)
    for sizes in ((511, 4096, 32000), (2000, 4096, 4095), (2000, 4096, 4088), (2000, 576, 32000), (600, 576, 49152), (700, 2048, 32768), (2000, 64, 1 << 20), (40000, 4096, 32000), (-1, 4096, 32000), (2000, -8, 32000),
                  (2000, 4096, -8), (1 << 31, 4096, 32000)):
        assert size(*sizes) == 0, sizes

    def bwd(x=4096, w=4096, t=4096, ms=4096, g=4096, dx=4096, dw=4096, M=2800, K=576, N=49152, ldw=576, T=1.0, ws=4096, bytes=1 << 30):
        P = ctypes.c_void_p
        return lib.pico_linear_log_probs_bwd(P(x), P(w), P(t), P(ms), P(g), P(dx), P(dw), M, K, N, ldw, T, -100, P(ws), bytes, None)
    for over in (dict(M=100), dict(M=0), dict(K=64), dict(N=4096), dict(ldw=568), dict(ldw=1 << 30), dict(T=0.0)):
        assert bwd(**over) == -3, over
    for over in (dict(x=4104), dict(w=4098), dict(t=4100), dict(ms=4100), dict(ws=4104), dict(dx=4104), dict(dw=4098)):
        assert bwd(**over) == -4, over
    for over in (dict(x=None), dict(w=None), dict(t=None), dict(ms=None), dict(g=None), dict(dx=None), dict(dw=None), dict(ws=None)):
        assert bwd(**over) == -1, over
    assert bwd(bytes=size(2800, 576, 49152) - 1) == -6 and "workspace" in message(lib)


def test_weight_gradient_of_few_rows(lib):
    def call(d=4096, x=4096, dw=4096, rows=8, out=100, inn=64, ldd=100, ldx=64):
        P = ctypes.c_void_p
        return lib.pico_weight_grad_few(P(d), P(x), P(dw), rows, out, inn, ldd, ldx, None)
    for over in (dict(rows=0), dict(rows=33), dict(out=0), dict(inn=0), dict(inn=60), dict(out=1 << 30), dict(inn=1 << 30)):
        assert call(**over) == -3, over
    for over in (dict(ldd=99), dict(ldx=63)):
        assert call(**over) == -5, over
    for over in (dict(d=None), dict(x=None), dict(dw=None)):
        assert call(**over) == -1, over
    for over in (dict(d=4097), dict(x=4097), dict(dw=4104)):
        assert call(**over) == -4, over


def test_host_path_refusals():
    """Tensors on the CPU are refused, not computed, and shapes are looked at first."""
    from picotron_amd.functional import linear_log_probs, log_probs, policy_loss, preference_loss
    x, t = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.long)
    for call in (lambda: linear_log_probs(x, torch.zeros(4, 8), t), lambda: log_probs(x, t), lambda: policy_loss(x, t, torch.zeros(2, 1)), lambda: preference_loss(x, t)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.mark.gpu
def test_host_path_refusals_on_the_gpu(device):
    from picotron_amd.functional import log_probs, policy_loss, preference_loss
    x = torch.zeros(2, 3, 8, device=device, dtype=torch.bfloat16)
    t = torch.zeros(2, 3, dtype=torch.long, device=device)
    A = torch.zeros(2, 1, device=device)

    def refused(match, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*args, **kw)
    for fn, rest in ((log_probs, ()), (policy_loss, (A,)), (preference_loss, ())):
        refused("one entry per row", fn, x, t[:, :2], *rest)
        refused("int64", fn, x, t.int(), *rest)
        refused("GPU only", fn, x, t.cpu(), *rest)
        refused("unit stride", fn, x.transpose(1, 2).contiguous().transpose(1, 2), t, *rest)
        refused("not supported", fn, x.half(), t, *rest)
        y = x.clone().requires_grad_()
        out = fn(y, t, *rest)
        out = out if torch.is_tensor(out) else out[0]
        refused("differentiated again", torch.autograd.grad, out.sum(), y, create_graph=True)
    refused("temperature", log_probs, x, t, temperature=0.0)
    refused("advantages", policy_loss, x, t, torch.zeros(3, 1, device=device))
    refused("advantages", policy_loss, x, t, torch.zeros(2, 1, dtype=torch.long, device=device))
    refused("GPU only", policy_loss, x, t, A.cpu())
    refused("old_log_probs", policy_loss, x, t, A, torch.zeros(2, 2, device=device))
    refused("ref_log_probs", policy_loss, x, t, A, kl_coef=0.1)
    refused("weights", policy_loss, x, t, A, weights=torch.zeros(5, device=device))
    refused("clip", policy_loss, x, t, A, clip=(-0.1, 0.2))
    refused("even", preference_loss, x[:1], t[:1])
    refused("2 pairs", preference_loss, x[0], t[0])
    refused("ref_log_probs", preference_loss, x, t, torch.zeros(3, device=device))
    refused("label_smoothing", preference_loss, x, t, label_smoothing=-0.1)


@pytest.mark.gpu
def test_targets_outside_the_vocabulary_can_be_checked(device, monkeypatch):
    from picotron_amd.functional import log_probs, policy_loss, preference_loss
    x = torch.zeros(2, 3, 8, device=device)
    t = torch.zeros(2, 3, dtype=torch.long, device=device)
    t[1, 1] = 8
    monkeypatch.setenv("PICO_CHECK_TARGETS", "1")
    for fn, rest in ((log_probs, ()), (policy_loss, (torch.zeros(2, 1, device=device),)), (preference_loss, ())):
        with pytest.raises(RuntimeError, match="1 targets lie outside"):
            fn(x, t, *rest)
