"""The fused linear layer, counter-based dropout and the loss without logits where values and calls are at their edges: numbers that are not
numbers, tails, certain answers, derivatives of other kinds, SM quotas.  u = 2^-8 is half a step of bfloat16."""
import gc
import math

import pytest
import torch

from tests.test_fused_training_gpu import BF, U, rng_of, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(built):
    from orion_b200 import torch_ops
    return torch_ops.load()


@pytest.fixture(autouse=True)
def status(built):
    yield
    from orion_b200 import kernels
    assert kernels.read_status() == 0


# few rows straight to registers and through the ring, tiles, a split reduction, odd widths of each
PATHS = [(3, 64, 64), (16, 20000, 512), (600, 1024, 4096), (600, 1023, 4096), (300, 1000, 2056), (2050, 520, 72), (130, 73, 136), (33, 250, 4104), (5, 257, 1024)]


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("M,N,K", PATHS)
def test_not_a_number_stays_one_behind_every_activation(ops, M, N, K, act):
    """A row of x, a row of w and an entry of the bias that are not numbers: every output that they reach is none either and the others are
    what they were; so with the gradients, whose dz is none there: rows of dx, rows of dw and entries of the bias's."""
    torch.manual_seed(M + N)
    x, w, b = torch.randn(M, K, device="cuda").to(BF), (torch.randn(N, K, device="cuda") / math.sqrt(K)).to(BF), torch.randn(N, device="cuda").to(BF)
    dy = torch.randn(M, N, device="cuda").to(BF)
    clean = ops.linear_act(x, w, b, None, act)
    row, col, entry = M // 2, N // 3, N - 1
    for what in ("x", "w", "bias"):
        bad = {"x": x.clone(), "w": w.clone(), "bias": b.clone()}
        bad[what][row if what == "x" else col if what == "w" else entry] = float("nan")
        hit = torch.zeros(M, N, dtype=torch.bool, device="cuda")
        hit[row if what == "x" else slice(None), slice(None) if what == "x" else col if what == "w" else entry] = True
        leaves = [bad[k].requires_grad_(True) for k in ("x", "w", "bias")]
        for y in (ops.linear_act(*(t.detach() for t in leaves), None, act), ops.linear_act(*leaves, None, act)):
            assert torch.equal(y.isnan(), hit) and torch.equal(y[~hit], clean[~hit])
        if act == "none":   # dz is dy, whatever z holds
            continue
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        rows, cols = hit.any(1), hit.any(0)
        assert dx[rows].isnan().all() and dw[cols].isnan().all() and torch.equal(db.isnan(), cols)
        if what == "bias":   # x and w are sound: nothing else is touched
            assert not dw[~cols].isnan().any()


def test_forward_mode_derivatives_are_refused(ops):
    """A tangent may not vanish: whichever argument carries one, in grad mode or not, the call is refused."""
    import torch.autograd.forward_ad as fw
    torch.manual_seed(1)
    x, w, b, r = (torch.randn(*s, device="cuda").to(BF) for s in ((8, 64), (16, 64), (16,), (8, 16)))
    target, rng = torch.zeros(8, dtype=torch.int64, device="cuda"), rng_of(1, 2)
    calls = [(lambda x, w, b, r: ops.linear_act(x, w, b, r, "gelu"), 4), (lambda x, w, b, r: ops.dropout(x, 0.5, rng), 1),
             (lambda x, w, b, r: ops.linear_cross_entropy(x, w, target), 2)]
    with fw.dual_level():
        for call, n in calls:
            for i in range(n):
                args = [x, w, b, r]
                args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="jvp|forward"):
                        call(*args)
    assert ops.linear_act(x, w, b, r, "gelu").shape == (8, 16)


@pytest.mark.parametrize("T", [3, 20, 100, 128, 300, 700])
@pytest.mark.parametrize("V", [200, 5003])
@pytest.mark.parametrize("base", [0.0, 8192.0, -8192.0])
def test_losses_next_to_large_logits_and_of_rows_that_are_sure(ops, T, V, base):
    """Logits that float32 holds exactly (multiples of 1/16 about `base`), so that only the loss's own arithmetic is off: of a weighted mean
    of V exponentials the exponents' rounding, 2^-24 of a distance to the maximum of at most some 15 where it weighs, 2^-22 of an
    exponential and some 40 float32 additions, 2^-18 in all, whatever the logits' size; and the result's rounding.  Half of the
    rows are sure: losses next to zero, none below it."""
    torch.manual_seed(V + T)
    H = 64
    w = (torch.randint(-8, 9, (V, H), device="cuda") / 16).to(BF)
    w[:, :16] = base / 16
    x = torch.ones(T, H, device="cuda").to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    # row t has the answer of its label's first free column: a unit 12 above there for the sure half
    x[:, 16:32] = 0
    w[:, 16:32] = 0
    label = torch.arange(0, T, 2, device="cuda")
    target[label] = V // 2
    w[V // 2, 16] = 24
    x[label, 16] = 1
    target[T // 2 + 1:T // 2 + 3] = -100
    counts = target != -100
    logits = x.double() @ w.double().T
    want = torch.where(counts, torch.logsumexp(logits, 1) - logits.gather(1, target.clamp(0)[:, None])[:, 0], 0.0)
    got = ops.linear_cross_entropy(x, w, target, reduction="none")
    within(got, want, 2.0 ** -18 + 2.0 ** -23 * want.abs(), "loss")
    assert (got >= 0).all()


@pytest.mark.parametrize("M,N", [(1, 8), (9, 16), (32, 8), (2000, 40), (2000, 33)])
def test_gelu_of_far_negative_values_is_relatively_exact(ops, M, N):
    """z is given exactly (a row of x with one entry, a column of ones), so that only GELU and the output's rounding are off: 0.16 % down to
    -5.6, 2.5 % of what is smaller than 6e-8 (fast_gelu.cuh), and half a step of bfloat16.  The slope, in float16: half a step
    relatively and 2^-25, and 3e-7 of the evaluation."""
    from orion_b200 import kernels as K
    z = -torch.logspace(-2, math.log10(12), M, device="cuda", dtype=torch.float64).to(BF)
    x, w = torch.zeros(M, 8, device="cuda", dtype=BF), torch.zeros(N, 8, device="cuda", dtype=BF)
    x[:, 0], w[:, 0] = z, 1
    zd = z.double()
    cdf = 0.5 * torch.special.erfc(-zd / math.sqrt(2))
    want = (zd * cdf)[:, None].expand(M, N)
    y, slope = K.linear_act(x, w, act="gelu", want_slope=True)
    bound = (U + torch.where(zd >= -5.6, 1.6e-3, 0.025))[:, None] * want.abs()
    for got in (y, ops.linear_act(x, w, act="gelu")):
        assert ((got.double() - want).abs() <= bound).all()
    s = (cdf + zd * torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi))[:, None].expand(M, N)
    within(slope[:, :N], s, 2.0 ** -11 * s.abs() + 2.0 ** -25 + 3e-7, "slope")


def test_a_gradient_of_the_residual_alone_keeps_no_slope(ops):
    """Memory of the call: the output alone; with a gradient of any other argument the slope, as large, beside it."""
    gc.collect()   # nothing of the tests before is freed in between
    torch.manual_seed(2)
    M, N, K = 512, 1024, 64
    x, w, b, r = torch.randn(M, K, device="cuda").to(BF), torch.randn(N, K, device="cuda").to(BF), torch.randn(N, device="cuda").to(BF), torch.randn(M, N, device="cuda").to(BF)
    dy = torch.randn(M, N, device="cuda").to(BF)
    want = ops.linear_act(x, w, b, r, "gelu")
    for i, copies in ((0, 2), (1, 2), (2, 2), (3, 1)):
        args = [t.detach().clone() for t in (x, w, b, r)]
        args[i].requires_grad_(True)
        before = torch.cuda.memory_allocated()
        y = ops.linear_act(*args, "gelu")
        assert torch.cuda.memory_allocated() - before == copies * M * N * 2
        assert torch.equal(y.detach(), want)
        g, = torch.autograd.grad(y, args[i], dy)
        assert g.shape == args[i].shape and (i < 3 or torch.equal(g, dy))
        del y, g


@pytest.fixture
def one_thread():
    """A quota belongs to the thread that sets it: backward passes in the calling thread, so that it holds for them too."""
    torch.autograd.set_multithreading_enabled(False)
    yield
    torch.autograd.set_multithreading_enabled(True)


def under_quotas(ops, quotas, run):
    want = run()
    for q in quotas:
        ops.set_sm_quota(q)
        got = run()
        ops.set_sm_quota(0)
        for a, b in zip(got, want):
            assert torch.equal(a, b), q


@pytest.mark.parametrize("M,N,K", [(16, 512, 512), (128, 520, 264), (300, 1000, 2056), (600, 1024, 4096), (2050, 520, 72), (1040, 73, 136), (33, 257, 1024)])
def test_gradients_of_the_layer_have_the_same_bits_from_any_cta_count(ops, one_thread, M, N, K):
    torch.manual_seed(M + K)
    x, w, b = torch.randn(M, K, device="cuda").to(BF), (torch.randn(N, K, device="cuda") / math.sqrt(K)).to(BF), torch.randn(N, device="cuda").to(BF)
    dy, rng = torch.randn(M, N, device="cuda").to(BF), rng_of(M, N)

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        return torch.autograd.grad(ops.linear_act(*leaves, None, "gelu", 0.1, rng, 4), leaves, dy)
    under_quotas(ops, (147, 31, 2, 1), run)


@pytest.mark.parametrize("T,V,H", [(12, 2000, 512), (128, 5003, 136), (700, 5003, 136), (1143, 9000, 768), (5000, 24001, 136)])
def test_gradients_of_the_loss_have_the_same_bits_from_any_cta_count(ops, one_thread, T, V, H):
    """All rows count, most, few: the gradient products are cut on the device for the rows that do."""
    torch.manual_seed(T + V)
    x, w = torch.randn(T, H, device="cuda").to(BF), (torch.randn(V, H, device="cuda") * 2 / math.sqrt(H)).to(BF)
    labels, out = torch.randint(0, V, (T,), device="cuda"), torch.randperm(T, device="cuda")
    for counted in sorted({T, T - T // 4, T // 7, 1, 0}):
        target = labels.clone()
        target[out[counted:]] = -100

        def run():
            leaves = [t.clone().requires_grad_(True) for t in (x, w)]
            loss = ops.linear_cross_entropy(*leaves, target)
            return [loss.detach()] + list(torch.autograd.grad(loss, leaves))
        under_quotas(ops, (147, 31, 2, 1), run)


FIRST_CALLS = r"""
import torch
from orion_b200 import torch_ops, kernels
ops = torch_ops.load()
BF = torch.bfloat16
randn = lambda *s: torch.randn(*s, device="cuda").to(BF)
x, few, w, t = randn(600, 512), randn(8, 512), randn(20000, 512).requires_grad_(True), torch.randint(0, 20000, (600,), device="cuda")
rng = torch.tensor([1, 2], device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):      # nothing of the library has run before
    out = [ops.linear_act(few, w, None, None, "gelu").detach(), ops.linear_act(x, w[:1024], None, None, "relu", 0.1, rng).detach(), ops.dropout(x, 0.2, rng)]
    loss = ops.linear_cross_entropy(x, w, t)
    out += [loss.detach()] + list(torch.autograd.grad(loss, w))
    del loss
graph.replay()
torch.cuda.synchronize()
want = [ops.linear_act(few, w, None, None, "gelu"), ops.linear_act(x, w[:1024], None, None, "relu", 0.1, rng), ops.dropout(x, 0.2, rng)]
loss = ops.linear_cross_entropy(x, w, t)
want += [loss] + list(torch.autograd.grad(loss, w))
assert all(torch.equal(a, b) for a, b in zip(out, want))
assert kernels.read_status() == 0
print("SAME")
"""


def test_the_first_call_of_a_process_may_be_captured(built):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "SAME" in run.stdout, run.stderr[-3000:]


def test_two_threads_train_at_once(ops):
    """Each with its own stream and quota: the results of a thread alone."""
    import threading

    def data(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
        return rn(600, 512), (rn(5003, 512).float() / 16).to(BF), rn(512, 512), torch.randint(0, 5003, (600,), device="cuda", generator=g)

    def step(x, w, u, t, seed):
        w, u = w.clone().requires_grad_(True), u.clone().requires_grad_(True)
        h = ops.linear_act(x, u, None, x, "gelu", 0.1, rng_of(seed, 1), 3)
        loss = ops.linear_cross_entropy(h, w, t)
        return [loss.detach()] + list(torch.autograd.grad(loss, (w, u)))
    inputs = [data(s) for s in range(2)]
    want = [step(*inputs[s], s) for s in range(2)]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def client(s):
        try:
            ops.set_sm_quota(40 + 60 * s)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(15):
                    got[s].append(step(*inputs[s], s))
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # shown in the test's thread
            errors.append(e)
    threads = [threading.Thread(target=client, args=(s,)) for s in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for s in range(2):
        for run in got[s]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[s]))


@pytest.mark.parametrize("M,N,K", [(8, 5000, 16384), (8, 5000, 16392), (40, 24, 40000), (1, 1, 8), (4097, 8, 8)])
def test_long_reductions_and_thin_layers(ops, M, N, K):
    """The ring's longest reduction, one piece more, a few-row launch of a reduction of any length, and the thinnest layer: bound as in
    the other tests (accumulation (K + 8) 2^-23 of the magnitudes)."""
    torch.manual_seed(K)
    x, w = torch.randn(M, K, device="cuda").to(BF), (torch.randn(N, K, device="cuda") / math.sqrt(K)).to(BF)
    z, mag = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    within(ops.linear_act(x, w), z, U * z.abs() + (K + 8) * 2.0 ** -23 * mag, "y")


def test_the_same_tensor_as_input_and_residual_and_everything_dropped(ops):
    torch.manual_seed(3)
    n = 136
    x, w, b = torch.randn(77, n, device="cuda").to(BF), torch.randn(n, n, device="cuda").to(BF), torch.randn(n, device="cuda").to(BF)
    dy, rng = torch.randn(77, n, device="cuda").to(BF), rng_of(1, 1)
    xs = x.clone().requires_grad_(True)
    y = ops.linear_act(xs, w, b, xs, "relu")
    a, r = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    y2 = ops.linear_act(a, w, b, r, "relu")
    ga, gr = torch.autograd.grad(y2, (a, r), dy)
    assert torch.equal(y, y2) and torch.equal(torch.autograd.grad(y, xs, dy)[0], ga + gr)
    # nothing is kept: the residual alone, and gradients of nothing
    for act in ("none", "gelu"):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b, x)]
        y = ops.linear_act(*leaves, act, 1.0, rng)
        assert torch.equal(y.detach(), x)
        dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
        assert not dx.any() and not dw.any() and not db.any() and torch.equal(dr, dy)


@pytest.mark.parametrize("M,N,K", [(16, 512, 512), (300, 1000, 2056), (2050, 520, 72), (130, 73, 136)])
def test_each_gradient_of_the_layer_alone(ops, M, N, K):
    """The bias's is the same; dx and dw may have their sums cut otherwise: each off by (terms + 8) 2^-23 of their magnitudes, |dz| <= 1.13 |dy|
    over the kept share, and by its rounding."""
    torch.manual_seed(M)
    x, w, b = torch.randn(M, K, device="cuda").to(BF), (torch.randn(N, K, device="cuda") / math.sqrt(K)).to(BF), torch.randn(N, device="cuda")
    dy, rng = torch.randn(M, N, device="cuda").to(BF), rng_of(M, N)

    def grads(want):
        leaves = [t.clone().requires_grad_(i in want) for i, t in enumerate((x, w, b))]
        y = ops.linear_act(*leaves, None, "gelu", 0.1, rng, 4)
        return dict(zip(want, torch.autograd.grad(y, [leaves[i] for i in want], dy)))
    together = grads((0, 1, 2))
    d = 1.13 / 0.89 * dy.double().abs()
    mags = ((N + 8) * 2.0 ** -23 * (d @ w.double().abs()), (M + 8) * 2.0 ** -23 * (d.T @ x.double().abs()))
    for want in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        for i, g in grads(want).items():
            if i == 2:
                assert torch.equal(g, together[2])
            else:
                within(g, together[i].double(), 2 * U * together[i].double().abs() + 2 * (1 + U) * mags[i], "xw"[i])


def test_a_captured_loss_of_few_rows_counts_them_anew(ops):
    """Up to 128 rows stay in place; which of them count is read at each replay."""
    T, V, H = 100, 3001, 72
    torch.manual_seed(4)
    x, w = torch.randn(T, H, device="cuda").to(BF).requires_grad_(True), (torch.randn(V, H, device="cuda") / 8).to(BF).requires_grad_(True)
    labels, target = torch.randint(0, V, (T,), device="cuda"), torch.zeros(T, device="cuda", dtype=torch.long)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(ops.linear_cross_entropy(x, w, target), (x, w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        loss = ops.linear_cross_entropy(x, w, target)
        out = [loss.detach()] + list(torch.autograd.grad(loss, (x, w)))
        del loss
    for counted in (100, 1, 0, 37, 100):
        target.copy_(labels)
        target[torch.randperm(T, device="cuda")[counted:]] = -100
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.linear_cross_entropy(x, w, target)
        want = [eager.detach()] + list(torch.autograd.grad(eager, (x, w)))
        assert all(torch.equal(a, b) for a, b in zip(out, want)), counted
        del eager
