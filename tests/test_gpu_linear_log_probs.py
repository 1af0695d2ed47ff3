"""Log-probabilities straight from hidden states and the vocabulary projection, against the definition in 64 bits, element by element.

Tolerances.  u = 2^-24.  A logit is a sum of hidden bf16 products, exact in fp32, added 32 at a time: off by at most Z = (hidden / 32 + 8) u sum
|x_k w_jk|.  A log-probability is off by two of them over T (its own and the weighted ones of the sum), by the exponentials' and the sum's
share, 2^-16 (V / 16 terms a thread's share at most joined over 32 slices), and 4 u of itself.  d(logits) is a ([j = t] - p_j) / T with p's relative error of
that and 2^-15, rounded to bf16 (2^-8 of itself); the two products with it are off by the sums of |d(logits) - exact| |w| (|x|), their own sums
(under 2^-10 of |d(logits)| |w|, contractions up to 49152) and one rounding to bf16.  What is under the smallest normal number, 2^-126, may be
taken for 0, p as well as d(logits) (p and a p / T each lose up to that, the latter a / T times the first): 2^-125 (1 + |a| / T) of every d(logits)."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
IGNORE = -100


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(seed, rows, hidden, vocab, kept=0.8, size=2.0):
    g = gen(seed)
    rows = rows if isinstance(rows, tuple) else (rows,)
    x = torch.randn(*rows, hidden, generator=g, device="cuda").to(BF16)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * (size / hidden ** 0.5)).to(BF16)
    t = torch.randint(0, vocab, rows, generator=g, device="cuda")
    t[torch.rand(rows, generator=g, device="cuda") >= kept] = IGNORE
    return x, w, t


def check(x, w, t, T=1.0, ignore=IGNORE, seed=0, grads=True):
    from picotron_amd.functional import linear_log_probs
    V, K = w.shape
    n = (t != ignore) & (t >= 0) & (t < V)
    xd, wd = x.detach().double().reshape(-1, K), w.detach().double()
    z = xd @ wd.t() / T
    Z = (K / 32 + 8) * 2 ** -24 * (xd.abs() @ wd.abs().t()).amax(1).view(t.shape) / T
    every = torch.log_softmax(z, -1)
    tt = t.clamp(0, V - 1).reshape(-1, 1)
    lp = torch.where(n, every.gather(1, tt).view(t.shape), 0.0)
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    with torch.no_grad():
        quiet = linear_log_probs(x, w, t, ignore, T)
    q = linear_log_probs(x, w, t, ignore, T)
    assert q.shape == t.shape and q.dtype == F32 and torch.equal(q, quiet)
    off = torch.where(n, 2 * Z + 2 ** -16 + 2 ** -22 * lp.abs(), 0.0)
    over = (q.double() - lp).abs() - off
    assert not q.isnan().any() and (over <= 0).all(), over.max().item()
    if not grads:
        return
    a = torch.randn(t.shape, generator=gen(seed + 5), device="cuda")
    ad = torch.where(n, a.double(), 0.0).view(-1, 1) / T
    p = every.exp()
    hot = torch.zeros_like(p).scatter_(1, tt, 1.0)
    d = ad * (hot - p)
    dd = 2 ** -125 * (1 + ad.abs()) + 2 ** -8 * d.abs() + ad.abs() * (p * (2 * Z.view(-1, 1) + 2 ** -15) + hot * 2 ** -21)
    dx, dw = torch.autograd.grad(q, (x, w), a, retain_graph=True)
    for got, want, bound in ((dx.reshape(-1, K), d @ wd, dd @ wd.abs() + 2 ** -10 * (d.abs() @ wd.abs())),
                             (dw, d.t() @ xd, dd.t() @ xd.abs() + 2 ** -10 * (d.abs().t() @ xd.abs()))):
        over = (got.double() - want).abs() - bound - 2 ** -8 * want.abs() - 1e-37
        assert got.dtype == BF16 and not got.isnan().any() and (over <= 0).all(), over.max().item()
    assert dx.shape == x.shape and dw.shape == w.shape


@pytest.mark.parametrize("rows,hidden,vocab", [(1, 72, 1), (1, 72, 8), (1, 128, 1000), (2, 96, 63), (3, 128, 64), (5, 128, 65), (7, 576, 49152), (64, 72, 257), (65, 200, 511),
                                               (128, 576, 1000), (129, 264, 1003), (257, 2048, 4099), (300, 1000, 32001), (513, 72, 66), (1000, 128, 777), (700, 136, 20000),
                                               (2049, 192, 4096), (90, 4096, 2500), (15, 584, 64), (16, 136, 1000), (17, 2048, 999), (32, 320, 4000), (33, 1096, 3000), (48, 264, 640),
                                               (49, 200, 127), (64, 4096, 2049)])
def test_over_sizes(device, rows, hidden, vocab):
    x, w, t = inputs(rows + hidden + vocab, rows, hidden, vocab)
    t[0], t[-1] = 0, vocab - 1
    check(x, w, t)
    check(x, w, t, T=0.7)


@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 383, 385, 511, 640, 1023])
def test_rows_at_the_ends_of_tiles(device, rows):
    """Every row's target in turn at the ends of the groups of 64 columns and of the tiles."""
    x, w, t = inputs(rows, rows, 128, 1029, kept=1.0)
    at = torch.tensor([0, 3, 4, 15, 16, 63, 64, 127, 128, 191, 192, 255, 256, 319, 511, 512, 767, 768, 1023, 1024, 1027, 1028], device="cuda")
    t.copy_(at[torch.arange(rows, device="cuda") % at.numel()])
    check(x, w, t)


def test_many_rounds_of_tiles(device):
    """More tiles than workgroups, of every height: the targets and rows of a tile arrive while the tile before leaves."""
    for rows, vocab in ((1100, 16500), (1500, 14000), (4096, 6000), (800, 30000)):
        x, w, t = inputs(rows, rows, 128, vocab)
        check(x, w, t)


@pytest.mark.parametrize("rows,vocab", [(1001, 16010), (190, 65001), (255, 49001), (510, 24501), (127, 65001), (130, 32003), (127, 48003)])
def test_every_shape_of_tile(device, rows, vocab):
    """Sizes that take 256 x 256, 192 x 256, 256 x 192, 128 x 256 and 128 x 192, whose waves have
    48 columns: targets at the ends of both widths, in the first and the last tile."""
    x, w, t = inputs(rows + vocab, rows, 96, vocab, kept=0.9)
    at = [k * n + d for n in (48, 64, 192, 256) for k in (0, 1, 2, 3, 4, (vocab - 1) // n) for d in (-1, 0, 1)] + [vocab - 1, vocab // 2]
    at = torch.tensor(sorted({c for c in at if 0 <= c < vocab}), device="cuda")
    t[::2] = at[torch.arange(t[::2].numel(), device="cuda") % at.numel()]
    check(x, w, t)


def test_strides(device):
    """Hidden states and weights with a row pitch, halves of wider buffers, rows that are no multiple of 16 bytes (copied), more axes, slices of tokens."""
    g = gen(1)
    wide = torch.randn(6, 50, 400, generator=g, device="cuda").to(BF16)
    big = (torch.randn(901, 400, generator=g, device="cuda") * 0.1).to(BF16)
    ids = torch.randint(0, 901, (6, 51), generator=g, device="cuda")
    check(wide[..., :200], big[:, 200:], ids[:, 1:])
    check(wide[:, ::2, 8:208], big[100:, :200], torch.where(ids[:, :50:2] < 801, ids[:, :50:2], IGNORE))
    check(wide[..., 3:203], big[:, 5:205], ids[:, 1:])
    check(wide.view(2, 3, 50, 400)[..., :200], big[:, :200], ids[:, 1:].reshape(2, 3, 50))
    check(wide[2, 3, :200], big[:, :200], ids[2, 3])
    flat = torch.randn(1 + 7 * 200, generator=g, device="cuda").to(BF16)
    check(flat[1:].view(7, 200), big[:, :200], ids[0, :7])          # rows without gaps that start beside a 16-byte boundary
    odd = torch.randn(5, 403, generator=g, device="cuda").to(BF16)
    check(odd[2:3, :200], big[:, :200], ids[0, :1])                  # one row, whose pitch does not matter
    check(odd[:, :200], big[4:5, :200], torch.zeros_like(ids[0, :5]))


def test_tokens_that_do_not_count(device):
    from picotron_amd.functional import linear_log_probs
    x, w, t = inputs(2, (4, 33), 128, 500, kept=1.0)
    t[0, 0], t[0, 1], t[0, 2], t[0, 3] = IGNORE, 500, -1, 2 ** 40 + 3
    check(x, w, t)
    check(x, w, t, ignore=int(t[1, 1]))
    y = x.clone()
    y[0, :4] = float("nan")
    q = linear_log_probs(y, w, t)
    assert not q[0, :4].any() and torch.equal(q, linear_log_probs(x, w, t))
    y, v = y.requires_grad_(), w.clone().requires_grad_()
    (dx,) = torch.autograd.grad(linear_log_probs(y, v, t), y, torch.ones_like(q))
    assert not dx[0, :4].any() and not dx.isnan().any()
    none = torch.full_like(t, IGNORE)
    xs = x.clone().requires_grad_()
    q = linear_log_probs(xs, v, none)
    dx, dw = torch.autograd.grad(q, (xs, v), torch.ones_like(q))
    assert not q.any() and not dx.any() and not dw.any()
    e = torch.empty(0, 7, 128, dtype=BF16, device="cuda").requires_grad_()
    q = linear_log_probs(e, v, torch.empty(0, 7, dtype=torch.long, device="cuda"))
    dx, dw = torch.autograd.grad(q.sum(), (e, v))
    assert q.shape == (0, 7) and dx.shape == e.shape and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("rows,hidden,vocab", [(1100, 264, 33001), (4096, 704, 12001), (511, 264, 49001), (17001, 4096, 2051)])
def test_rows_that_do_not_count_change_nothing(device, rows, hidden, vocab):
    """Several rounds of tiles, where the rows that count are put together: the others hold NaN, and what counts gets the same bits whichever they are."""
    from picotron_amd.functional import linear_log_probs
    x, w, t = inputs(rows, rows, hidden, vocab, kept=1.0)
    every = linear_log_probs(x, w, t)
    check(x, w, t, grads=False)
    kept = torch.rand(rows, generator=gen(8), device="cuda")
    r = torch.arange(rows, device="cuda")
    for i, counts in enumerate((kept < 0.3, kept < 0.9, r >= rows // 2, r < rows // 2, (r // 100) % 3 == 1, r == 0, r == rows - 1, r < 0, r != 77, r > -1)):
        u = torch.where(counts, t, torch.where(r % 3 == 0, IGNORE, torch.where(r % 3 == 1, vocab, -1 - r)))
        y = torch.where(counts[:, None], x, float("nan"))
        assert torch.equal(linear_log_probs(y, w, u), torch.where(counts, every, 0.0)), i
    u, x = torch.where(kept < 0.3, t, IGNORE), x.requires_grad_()
    v = w.clone().requires_grad_()
    a = torch.randn(rows, generator=gen(9), device="cuda")
    dx, dw = torch.autograd.grad(linear_log_probs(x, v, u), (x, v), a)
    ex, ew = torch.autograd.grad(linear_log_probs(x, v, t), (x, v), torch.where(kept < 0.3, a, 0.0))
    assert torch.equal(dx, ex) and torch.equal(dw, ew) and not dx[kept >= 0.3].any()


@pytest.mark.parametrize("rows,hidden,vocab", [(2800, 576, 49152), (2000, 4096, 8192), (1503, 2048, 16392), (2049, 1000, 32776), (4100, 264, 65544), (512, 4096, 8200), (2000, 4096, 8191), (1503, 2048, 16385),
                                               (2800, 576, 49155)])
def test_gradients_of_the_rows_that_count(device, rows, hidden, vocab):
    """Sizes whose backward leaves out what does not count: against the definition, and the same bits whatever the other rows hold."""
    from picotron_amd import _lib
    from picotron_amd.functional import linear_log_probs
    assert _lib.lib().pico_linear_log_probs_bwd_workspace_bytes(rows, hidden, vocab) > 0
    x, w, t = inputs(rows, rows, hidden, vocab, kept=1.0)
    kept, r = torch.rand(rows, generator=gen(8), device="cuda"), torch.arange(rows, device="cuda")
    a = torch.randn(rows, generator=gen(9), device="cuda")
    for i, counts in enumerate((kept < 0.3, r < 0, r == rows - 3, r < 127, r >= rows - 129, (r // 100) % 3 == 1, kept < 0.9, r > -1)):
        u = torch.where(counts, t, IGNORE)
        if i in (0, 2, 3, 6, 7):
            check(x, w, u, seed=i)
        got = []
        for y in (x, torch.where(counts[:, None], x, float("nan"))):
            y, v = y.detach().clone().requires_grad_(), w.clone().requires_grad_()
            got.append(torch.autograd.grad(linear_log_probs(y, v, u), (y, v), torch.where(counts, a, float("inf"))))
        (dx, dw), (ex, ew) = got
        assert torch.equal(dx, ex) and torch.equal(dw, ew) and not dw.isnan().any() and not dx[~counts].any(), i
        assert dx[counts].any(1).all() and bool(dw.any()) == bool(counts.any()), i


def test_a_recorded_step_takes_other_rows_on_every_replay(device):
    from picotron_amd.functional import linear_log_probs
    x, w, t = inputs(5, 2049, 1000, 32776, kept=1.0)
    kept = torch.rand(2049, generator=gen(6), device="cuda")
    masked = [torch.where(kept < share, t, IGNORE) for share in (0.0, 0.5, 1.0, 0.04)]
    a = torch.randn(2049, generator=gen(7), device="cuda")

    def step(u):
        y, v = x.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(linear_log_probs(y, v, u), (y, v), a)
    want = [step(u) for u in masked]
    still = t.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        step(still)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(still)
    for i in (2, 0, 1, 3, 2, 1):
        still.copy_(masked[i])
        graph.replay()
        step(masked[(i + 1) % 4])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1]), i


@pytest.mark.parametrize("rows,hidden,vocab", [(1, 2048, 49152), (4, 2112, 49152), (16, 2048, 32000), (31, 1032, 60001), (32, 2048, 49151), (17, 4096, 20003),
                                               (33, 2112, 32000), (65, 4096, 10000), (100, 2112, 49152), (127, 4096, 32000), (127, 4096, 32001)])
def test_gradients_of_few_rows(device, rows, hidden, vocab):
    x, w, t = inputs(rows, rows, hidden, vocab, kept=1.0)
    check(x, w, t)
    t[rows // 2] = IGNORE
    check(x, w, t, T=0.8)


def test_weight_gradient_of_few_rows(device):
    """pico_weight_grad_few over rows, edges of its tiles and pitches: a sum of 32 exact products in fp32 (32 half steps of 2^-24 of their magnitudes) and one
    rounding, and not a byte behind dw."""
    import ctypes
    from picotron_amd import _lib
    lib, P = _lib.lib(), lambda v: ctypes.c_void_p(v.data_ptr())
    for rows, out, inn in ((1, 1, 8), (2, 15, 16), (7, 16, 24), (8, 17, 120), (9, 255, 128), (15, 256, 136), (16, 257, 512), (17, 300, 520), (31, 1000, 1032), (32, 513, 640), (32, 16, 2048)):
        g = gen(rows)
        d = torch.randn(rows, out + 3, generator=g, device="cuda").to(BF16)[:, :out]
        x = torch.randn(rows, inn + 5, generator=g, device="cuda").to(BF16)[:, 2:2 + inn]
        dw = torch.full((out * inn + 64,), 7.0, dtype=BF16, device="cuda")
        assert lib.pico_weight_grad_few(P(d), P(x), P(dw), rows, out, inn, d.stride(0), x.stride(0), None) == 0
        torch.cuda.synchronize()
        got, want = dw[:out * inn].view(out, inn).double(), d.double().t() @ x.double()
        over = (got - want).abs() - 2 ** -8 * want.abs() - 2 ** -18 * (d.double().abs().t() @ x.double().abs())
        assert (over <= 0).all() and (dw[out * inn:] == 7).all(), (rows, out, inn, over.max().item())


def test_a_recorded_call_takes_other_rows_on_every_replay(device):
    from picotron_amd.functional import linear_log_probs
    x, w, t = inputs(5, 1100, 264, 33001, kept=1.0)
    kept = torch.rand(1100, generator=gen(6), device="cuda")
    masked = [torch.where(kept < share, t, IGNORE) for share in (0.0, 0.5, 1.0, 0.2)]
    want = [linear_log_probs(x, w, u) for u in masked]
    still = t.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        linear_log_probs(x, w, still)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = linear_log_probs(x, w, still)
    for i in (2, 0, 1, 3, 2, 1):
        still.copy_(masked[i])
        graph.replay()
        linear_log_probs(x, w, masked[(i + 1) % 4])
        torch.cuda.synchronize()
        assert torch.equal(q, want[i]), i


def test_large_and_certain_logits(device):
    """Logits of several hundred, one token nearly certain in every row."""
    x, w, t = inputs(3, 200, 256, 3001, kept=1.0, size=30.0)
    check(x, w, t)
    w[t] = x * 0.05
    check(x, w, t)
    check(x, w, t, T=0.3)


def test_only_one_gradient_wanted_and_refusals(device):
    from picotron_amd.functional import linear_log_probs
    x, w, t = inputs(4, (2, 40), 128, 600)
    a = torch.randn(2, 40, device="cuda")
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(linear_log_probs(xs, ws, t), (xs, ws), a)
    for got, want in ((torch.autograd.grad(linear_log_probs(xs, w, t), xs, a)[0], dx), (torch.autograd.grad(linear_log_probs(x, ws, t), ws, a)[0], dw)):
        assert ((got.float() - want.float()).norm() / want.float().norm()).item() <= 2 ** -8      # (another product may take it)

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            linear_log_probs(*args, **kw)
    refused("one entry per row", x, w, t[:, :3])
    refused("int64", x, w, t.int())
    refused("bf16", x.float(), w, t)
    refused("bf16", x, w.float(), t)
    refused("weight must be", x, w[:, :120], t)
    refused("weight must be", x, w[0], t)
    refused("hidden a multiple of 8", x[..., :64], w[:, :64], t)
    refused("hidden a multiple of 8", x[..., :100], w[:, :100], t)
    refused("temperature", x, w, t, temperature=-1.0)
    refused("GPU only", x, w.cpu(), t)
    q = linear_log_probs(xs, ws, t)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(q.sum(), xs, create_graph=True)


@pytest.mark.parametrize("rows,hidden,vocab", [(200, 256, 5000), (700, 1000, 32777), (5, 2112, 20000)])
def test_streams_threads_and_graphs(device, rows, hidden, vocab):
    from picotron_amd.functional import linear_log_probs
    ready = [inputs(s, (3, rows), hidden, vocab, kept=(0.8, 1.0, 0.3)[s]) for s in range(3)]
    up = torch.randn(3, rows, generator=gen(9), device="cuda")

    def run(x, w, t):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        q = linear_log_probs(x, w, t)
        return (q.detach(), *torch.autograd.grad(q, (x, w), up))
    want = [run(*r) for r in ready]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [torch.zeros_like(v) for v in ready[0]]
        torch.cuda._sleep(3_000_000)
        for a, b in zip(late, ready[0]):
            a.copy_(b)
        got = run(*late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    mine = run(*(v.clone() for v in ready[i]))
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(mine, want[i])):
                        failed.append(i)
        except Exception as e:      # noqa: BLE001 (reported by the test's own thread)
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(timeout=100)
    assert not failed and not any(th.is_alive() for th in threads), failed
    still = [v.clone() for v in ready[0]]
    with torch.cuda.stream(side):
        run(*still)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*still)
    for i in (1, 2, 0, 1):
        for a, b in zip(still, ready[i]):
            a.copy_(b)
        graph.replay()
        run(*ready[(i + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i


def test_a_model_scores_its_tokens(device):
    """Llama.log_probs against log_probs of the model's own logits (which are rounded to bf16: 2^-8 of each), with gradients, and the reference of
    a preference step from it."""
    import picotron_amd.process_group_manager as pgm
    from picotron_amd.functional import log_probs, preference_loss
    from picotron_amd.model import Llama
    from picotron_amd.utils import ModelShape
    pgm.setup_process_group_manager(1, 1, 1, 1)
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = Llama(ModelShape(128, 2, 1, 256, 1000, 2, 64)).to(BF16)
    ids = torch.randint(0, 1000, (4, 65), generator=gen(1), device="cuda")
    t = ids[:, 1:].clone()
    t[:, :9] = IGNORE
    logits = model(input_ids=ids[:, :-1])
    want = log_probs(logits, t)
    got = model.log_probs(ids[:, :-1], t)
    assert (got - want).abs().max().item() <= 2 * 2 ** -8 * logits.abs().max().item()
    a = torch.randn(4, 64, generator=gen(2), device="cuda")
    params = list(model.parameters())
    for x, y in zip(torch.autograd.grad(want, params, a), torch.autograd.grad(got, params, a)):
        assert ((x.float() - y.float()).norm() / x.float().norm().clamp_min(1e-20)).item() <= 3e-2
    with torch.no_grad():
        ref = model.log_probs(ids[:, :-1], t)
        assert torch.equal(ref, got)
        loss, seq = preference_loss(model(input_ids=ids[:, :-1]), t, ref.sum(1))
    # the same policy and reference: x is 0 but for the logits' rounding
    assert abs(loss.item() - 0.693147) <= 0.1 * 55 * 2 * 2 ** -8 * logits.abs().max().item()
    assert (model.log_probs(ids[:, :-1], t, temperature=2.0)[:, 20] - log_probs(logits, t, temperature=2.0)[:, 20]).abs().max().item() <= 2 ** -8 * logits.abs().max().item()
    with_bias = type(model.final_proj)(128, 1000, bias=True).to("cuda", BF16)
    h = model.hidden_states(ids[:, :-1])
    assert torch.equal(with_bias.log_probs(h, t), log_probs(with_bias(h), t))
    for hidden in (64, 100):      # what the kernels for hidden states do not take
        small = type(model.final_proj)(hidden, 1000, bias=False).to("cuda", BF16)
        h = torch.randn(4, 64, hidden, generator=gen(3), device="cuda").to(BF16)
        assert torch.equal(small.log_probs(h, t), log_probs(small(h), t))
