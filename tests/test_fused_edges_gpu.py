"""The fused linear layer, counter-based dropout and the loss without logits where values and calls are at their edges: numbers that are not
numbers, tails, certain answers, derivatives of other kinds, SM quotas.  u = 2^-8 is half a step of bfloat16."""
import math

import pytest
import torch

from tests.test_fused_training_gpu import BF, U, act64, rng_of, within

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
