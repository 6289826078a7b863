"""The fused linear layer, counter-based dropout and the loss without logits against float64, element by element.

Where the bounds come from.  u = 2^-8 is half a step of bfloat16: an output rounded once is off by at most u of itself.  A float32
accumulation of K products is taken to be off by at most (K + 8) 2^-23 of the sum of their magnitudes (twice the textbook bound: the
tensor core's adder may cut where a float addition rounds).  GELU's CDF is off by 1.5e-7 (fast_gelu.cuh), exponentials and logarithms by
2^-20 of themselves.  The rest is first-order propagation, with a factor 1.01 for second-order terms."""
import math

import pytest
import torch

from tests.test_fused_training_host import plain_bits

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
BF = torch.bfloat16


def acc(k):
    return (k + 8) * 2.0 ** -23


@pytest.fixture(scope="module")
def ops(built):
    from orion_b200 import torch_ops
    return torch_ops.load()


@pytest.fixture(autouse=True)
def status(built):
    yield
    from orion_b200 import kernels
    assert kernels.read_status() == 0


def rng_of(seed, step):
    return torch.tensor([seed, step], dtype=torch.int64, device="cuda")


def keep_mask(n, p, rng, site):
    """(mask, factor) of n elements in int64 arithmetic on the GPU."""
    low, thr = 0xFFFFFFFF, min(65536, int(p * 65536 + 0.5))
    g = torch.arange((n + 7) // 8, device="cuda")
    c = [g & low, g >> 32 & 0xFFFF | (rng[1] >> 32 & 0xFFFF) << 16, (rng[1] & low).expand_as(g), torch.full_like(g, site)]
    k = [rng[0] & low, rng[0] >> 32 & low]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 & low ^ c[1] ^ k[0], b & low, a >> 32 & low ^ c[3] ^ k[1], a & low]
        k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
    w = torch.stack(c, 1)
    halves = torch.stack((w & 0xFFFF, w >> 16), 2).flatten()[:n]
    return halves >= thr, 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound * 1.01 + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), float((off / (bound + 1e-30)).max()))


def act64(z, act):
    """act(z), its derivative, and how far a float32 evaluation is off."""
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), z.abs() * 3e-7
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    return z, torch.ones_like(z), 0.0


def make(M, N, K, residual, bias_dtype, seed):
    torch.manual_seed(seed)
    x, w = torch.randn(M, K, device="cuda").to(BF), (torch.randn(N, K, device="cuda") / math.sqrt(K)).to(BF)
    b = torch.randn(N, device="cuda").to(bias_dtype) if bias_dtype else None
    r = torch.randn(M, N, device="cuda").to(BF) if residual else None
    return x, w, b, r


def expect(x, w, b, r, act, p, rng, site):
    """float64 output and its bound, and what the backward pass needs."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.T + (b.double() if b is not None else 0)
    mag = xd.abs() @ wd.abs().T + (b.double().abs() if b is not None else 0)
    dz_err = acc(x.shape[1]) * mag
    a, slope, eval_err = act64(z, act)
    a_err = dz_err * 1.13 + eval_err     # no activation here is steeper than 1.13
    keep, f = (keep_mask(z.numel(), p, rng, site) if p > 0 else (None, 1.0))
    m = keep.view(z.shape).double() * f if keep is not None else torch.ones_like(z)
    y = a * m + (r.double() if r is not None else 0)
    # float32: the scaled value and the sum are each rounded once more
    return y, U * y.abs() + a_err * m + 2.0 ** -23 * ((a * m).abs() + y.abs()), z, slope, m, dz_err


SIZES = [(1, 64, 64), (3, 8, 8), (16, 1024, 512), (77, 768, 768), (130, 72, 136), (17, 1, 64), (129, 33, 200), (5, 257, 1024), (33, 250, 72),
         (300, 1000, 2056), (64, 1024, 4096), (600, 1024, 4096), (2050, 520, 72), (4100, 1032, 136)]


@pytest.mark.parametrize("act,residual,p,bias", [("none", True, 0.0, BF), ("gelu", False, 0.0, torch.float32), ("gelu", True, 0.1, BF),
                                                 ("relu", True, 0.25, None), ("none", False, 0.5, torch.float32)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_act_forward(ops, M, N, K, act, residual, p, bias):
    x, w, b, r = make(M, N, K, residual, bias, M + N + K)
    rng = rng_of(0x1234567890ABCD + M, 2 ** 33 + N)
    want, bound = expect(x, w, b, r, act, p, rng, 5)[:2]
    y = ops.linear_act(x, w, b, r, act, p, rng, 5)
    within(y, want, bound, "y")
    # the same from any CTA count, and under grad mode, where the activation's slope is written beside it
    for n in (7, 1):
        ops.set_sm_quota(n)
        again = ops.linear_act(x, w, b, r, act, p, rng, 5)
        ops.set_sm_quota(0)
        assert torch.equal(again, y)
    assert torch.equal(ops.linear_act(x.requires_grad_(True), w, b, r, act, p, rng, 5).detach(), y)


@pytest.mark.parametrize("act,residual,p,bias", [("none", True, 0.0, BF), ("gelu", False, 0.0, torch.float32), ("gelu", True, 0.1, BF),
                                                 ("relu", True, 0.25, None), ("none", False, 0.5, torch.float32)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_act_gradients(ops, M, N, K, act, residual, p, bias):
    x, w, b, r = make(M, N, K, residual, bias, M + N + K)
    rng = rng_of(M, N)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    dy = torch.randn(M, N, device="cuda").to(BF)
    got = list(torch.autograd.grad(ops.linear_act(x, w, b, r, act, p, rng, 9), leaves, dy))
    with torch.no_grad():
        _, _, z, slope, m, z_err = expect(x, w, b, r, act, p, rng, 9)
        g = dy.double() * m
        dz = g * slope
        # the slope is kept in float16 (half a step 2^-11, absolute below 2^-14), taken at a float32 z: |gelu''| <= 0.8; near 0 a ReLU may
        # fall on the other side; only what a slope multiplied is rounded again
        if act == "gelu":
            dz_err = g.abs() * (2.0 ** -11 * slope.abs() + 2.0 ** -25 + 0.8 * z_err + 1e-6) + U * dz.abs()
        elif act == "relu":
            dz_err = torch.where(z.abs() <= 2 * z_err, g.abs(), 0.0)
        else:
            dz_err = torch.zeros_like(dz)
        dz_err = dz_err + 2.0 ** -22 * dz.abs()
        xd, wd = x.double(), w.double()
        want = dz @ wd
        within(got.pop(0), want, U * want.abs() + dz_err @ wd.abs() + acc(N) * (dz.abs() @ wd.abs()), "dx")
        want = dz.T @ xd
        within(got.pop(0), want, U * want.abs() + dz_err.T @ xd.abs() + acc(M) * (dz.abs().T @ xd.abs()), "dw")
        if b is not None:
            want, out = dz.sum(0), got.pop(0)
            assert out.dtype == b.dtype
            half = U if b.dtype == BF else 2.0 ** -24
            # summed before dz is rounded
            within(out, want, half * want.abs() + (dz_err - U * dz.abs() * (act == "gelu")).clamp(min=0).sum(0) + acc(M) * dz.abs().sum(0), "db")
        if r is not None:
            assert torch.equal(got.pop(0), dy)


@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("N,K", [(20000, 512), (20003, 1000), (2500, 4096), (1000, 5000), (9000, 40), (7, 8)])
def test_linear_act_of_few_rows(ops, M, N, K):
    """Single tokens: tiles of 8 and 16 rows of w, one and many of them for a CTA (the rings come round), reductions of one piece and
    of several, ragged ends of each; the same bits from any CTA count."""
    x, w, b, r = make(M, N, K, True, BF, M + N)
    rng = rng_of(5, 6)
    want, bound = expect(x, w, b, r, "gelu", 0.1, rng, 2)[:2]
    y = ops.linear_act(x, w, b, r, "gelu", 0.1, rng, 2)
    within(y, want, bound, "y")
    for q in (100, 3):
        ops.set_sm_quota(q)
        again = ops.linear_act(x, w, b, r, "gelu", 0.1, rng, 2)
        ops.set_sm_quota(0)
        assert torch.equal(again, y)
    # what a row of x holds beyond the others' concerns it alone
    bad = x.clone()
    bad[0] = float("nan")
    y2 = ops.linear_act(bad, w, b, r)
    assert y2[0].isnan().all() and torch.equal(y2[1:], ops.linear_act(x, w, b, r)[1:])


@pytest.mark.parametrize("T", [1, 8, 13, 32])
@pytest.mark.parametrize("V,H", [(32000, 1024), (20003, 200), (5000, 1536)])
def test_loss_of_few_rows(ops, T, V, H):
    torch.manual_seed(T + V)
    x, w = torch.randn(T, H, device="cuda").to(BF), (torch.randn(V, H, device="cuda") * 2 / math.sqrt(H)).to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    target[0] = V - 1
    out, _, _ = check_loss(ops, x, w, target, "none")
    ops.set_sm_quota(5)
    again = ops.linear_cross_entropy(x, w, target, reduction="none")
    ops.set_sm_quota(0)
    assert torch.equal(again, out)


def test_linear_act_gradient_is_the_difference_quotient(ops):
    """f(w) = sum(y * dy) along d: without an activation f is linear, so the quotient over any step is the derivative; with GELU the
    remainder of the central quotient is h^2 / 6 of the third derivative, |gelu'''| <= 2.4.  Steps and values have few bits, so that
    w +- h d are exact."""
    torch.manual_seed(0)
    M, N, K, h = 64, 40, 72, 0.25
    x = torch.randint(-8, 9, (M, K), device="cuda").to(BF) / 16
    w, d = torch.randint(-4, 5, (N, K), device="cuda").to(BF) / 8, torch.randint(-1, 2, (N, K), device="cuda").to(BF) / 4
    dy, rng = torch.randn(M, N, device="cuda").to(BF), rng_of(1, 2)
    for act, third in (("none", 0.0), ("gelu", 2.4)):
        wl = w.clone().requires_grad_(True)
        grad, = torch.autograd.grad(ops.linear_act(x, wl, None, None, act, 0.25, rng, 1), wl, dy)
        up, down = (ops.linear_act(x, w + s * h * d, None, None, act, 0.25, rng, 1).double() for s in (1, -1))
        quotient = ((up - down) * dy.double()).sum() / (2 * h)
        rounding = (U * (up.abs() + down.abs()) * dy.double().abs()).sum() / (2 * h)
        along = (x.double() @ d.double().T).abs()
        remainder = (dy.double().abs() * 1.34 * third * (along * h) ** 3 / 6 / h).sum()
        derivative = (grad.double() * d.double()).sum()
        assert abs(quotient - derivative) <= rounding + remainder + (2 * U * grad.double().abs() * d.double().abs()).sum() + 1e-3 * abs(derivative)


def test_linear_act_takes_any_layout_and_leading_dimensions(ops):
    torch.manual_seed(4)
    big = torch.randn(5, 9, 160, device="cuda").to(BF)
    w = torch.randn(48, 64, device="cuda").to(BF)
    wide = torch.randn(48, 136, device="cuda").to(BF)
    res = torch.randn(9, 5, 48, device="cuda").to(BF)
    for x in (big[:, :, :64], big[:, :, 3:67], big[:, :, 8:72].transpose(0, 1), big[1:2, :1, :64], big[:, ::2, 96:], big[0, 0, :64].expand(5, 9, 64)):
        for weight in (w, wide[:, 8:72], wide[:, 5:69], wide.T[:64].T, w.T.contiguous().T):
            for r in (None, res.transpose(0, 1)[: x.shape[0], : x.shape[1]] if x.shape[0] <= 5 and x.shape[1] <= 9 else None):
                a, b = x.detach().requires_grad_(True), weight.detach().requires_grad_(True)
                y = ops.linear_act(a, b, None, r)
                ac, bc = x.contiguous().requires_grad_(True), weight.contiguous().requires_grad_(True)
                yc = ops.linear_act(ac, bc, None, None if r is None else r.contiguous())
                assert y.shape == x.shape[:-1] + (48,) and y.is_contiguous() and torch.equal(y, yc)
                dy = torch.randn(48, *y.shape[:-1], device="cuda").to(BF).movedim(0, -1)
                for g, gc in zip(torch.autograd.grad(y, (a, b), dy), torch.autograd.grad(yc, (ac, bc), dy.contiguous())):
                    assert torch.equal(g, gc)
    # an upstream gradient that is one number for all, as sum().backward() gives
    a = big[:, :, :64].detach().requires_grad_(True)
    ops.linear_act(a, w).sum().backward()
    assert a.grad.shape == a.shape
    want = w.double().sum(0).expand(5, 9, 64)
    within(a.grad, want, U * want.abs() + acc(48) * w.double().abs().sum(0), "dx of a sum")


def test_linear_act_of_nothing(ops):
    w, b = (torch.randn(16, 8, device="cuda").to(BF).requires_grad_(True), torch.randn(16, device="cuda").to(BF).requires_grad_(True))
    x = torch.empty(0, 8, device="cuda", dtype=BF, requires_grad=True)
    y = ops.linear_act(x, w, b, None, "gelu", 0.1, rng_of(1, 1))
    assert y.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 8) and not w.grad.any() and not b.grad.any()
    assert ops.linear_act(torch.randn(3, 8, device="cuda").to(BF), torch.empty(0, 8, device="cuda", dtype=BF)).shape == (3, 0)


def test_operators_refuse_what_they_cannot_do(ops):
    x, w, rng = torch.randn(4, 8, device="cuda").to(BF), torch.randn(16, 8, device="cuda").to(BF), rng_of(1, 1)
    for bad in (lambda: ops.linear_act(x, w[:, :7]), lambda: ops.linear_act(x.float(), w), lambda: ops.linear_act(x, w.float()),
                lambda: ops.linear_act(x[0], w), lambda: ops.linear_act(x[:, :4], w[:, :4]), lambda: ops.linear_act(x, w, act="tanh"),
                lambda: ops.linear_act(x, w, torch.zeros(15, device="cuda")), lambda: ops.linear_act(x, w, torch.zeros(16)),
                lambda: ops.linear_act(x, w, torch.zeros(32, device="cuda")[::2]), lambda: ops.linear_act(x, w, None, torch.zeros(4, 8, device="cuda").to(BF)),
                lambda: ops.linear_act(x, w, None, torch.zeros(1, 16, device="cuda").to(BF)), lambda: ops.linear_act(x, w, p=0.1),
                lambda: ops.linear_act(x, w, p=1.5, rng=rng), lambda: ops.linear_act(x, w, p=float("nan"), rng=rng),
                lambda: ops.linear_act(x, w, p=0.1, rng=rng.cpu()), lambda: ops.linear_act(x, w, p=0.1, rng=rng.int()),
                lambda: ops.linear_act(x, w, p=0.1, rng=rng[:1]), lambda: ops.linear_act(x, w, p=0.1, rng=rng, site=-1),
                lambda: ops.linear_act(x, w.cpu()),
                lambda: ops.dropout(x.half(), 0.1, rng), lambda: ops.dropout(x, 0.1, None), lambda: ops.dropout(x, -0.1, rng),
                lambda: ops.dropout(x, 0.1, rng, 0, x.float()), lambda: ops.dropout(x, 0.1, rng, 0, x[:2]), lambda: ops.dropout(x, 0.1, rng, 2 ** 31),
                lambda: ops.linear_cross_entropy(x, w, torch.zeros(3, dtype=torch.int64, device="cuda")),
                lambda: ops.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int32, device="cuda")),
                lambda: ops.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64)), lambda: ops.linear_cross_entropy(x, w[:0], torch.zeros(4, dtype=torch.int64, device="cuda")),
                lambda: ops.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64, device="cuda"), reduction="max"),
                lambda: ops.linear_cross_entropy(x.float(), w, torch.zeros(4, dtype=torch.int64, device="cuda")),
                lambda: ops.linear_cross_entropy(x[:, :4], w[:, :4], torch.zeros(4, dtype=torch.int64, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()


# ------------------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 77 * 768, 4096 * 257 + 3])
@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 1.0])
def test_dropout_and_its_gradient(ops, n, p, dtype):
    torch.manual_seed(n)
    rng = rng_of(-5 - n, 3)   # a seed with its sign bit set
    x, r, dy = (torch.randn(n, device="cuda").to(dtype) for _ in range(3))
    keep, f = keep_mask(n, p, rng, 2)
    half = U if dtype == BF else 2.0 ** -24
    for res in (None, r):
        xl = x.clone().requires_grad_(True)
        y = ops.dropout(xl, p, rng, 2, res)
        a = torch.where(keep, x.double() * f, 0.0)
        want = a + (res.double() if res is not None else 0)
        within(y.detach(), want, half * want.abs() + 2.0 ** -23 * (a.abs() + want.abs()), "y")
        dx, = torch.autograd.grad(y, xl, dy)
        want = torch.where(keep, dy.double() * f, 0.0)
        within(dx, want, (half + 2.0 ** -23) * want.abs(), "dx")
        assert torch.equal(dx == 0, ~keep | (dy == 0))
    if p == 0.0:
        assert torch.equal(ops.dropout(x, 0.0, None), x)


def test_dropout_views_order_and_residual_gradient(ops):
    torch.manual_seed(1)
    base, rng = torch.randn(40, 67, device="cuda").to(BF), rng_of(3, 4)
    for x in (base[1:], base.T, base[:, 1:9], base.flatten()[3:1003], base[:, :1]):
        r = torch.randn(x.shape[::-1], device="cuda").to(BF).permute(*range(x.dim())[::-1])
        xl, rl = x.detach().requires_grad_(True), r.detach().requires_grad_(True)
        y = ops.dropout(xl, 0.3, rng, 0, rl)
        assert torch.equal(y, ops.dropout(x.contiguous(), 0.3, rng, 0, r.contiguous()))
        dy = torch.randn(x.shape[::-1], device="cuda").to(BF).permute(*range(x.dim())[::-1])
        dx, dr = torch.autograd.grad(y, (xl, rl), dy)
        assert torch.equal(dx, ops.dropout(dy.contiguous(), 0.3, rng, 0)) and torch.equal(dr, dy)
    # dropped elements are taken away, whatever they hold; those that are kept stay what they are
    bad = torch.full((1000,), float("nan"), device="cuda")
    keep, _ = keep_mask(1000, 0.5, rng, 0)
    y = ops.dropout(bad, 0.5, rng, 0)
    assert torch.equal(y.isnan(), keep) and not y[~keep].any()
    assert not ops.dropout(bad, 1.0, rng, 0).any()


def test_masks_keep_their_share_and_differ_by_step_site_and_seed(ops):
    n, p = 1 << 22, 0.1
    one = torch.ones(n, device="cuda")
    masks = [ops.dropout(one, p, rng_of(s, t), site) != 0 for s, t, site in ((1, 1, 1), (2, 1, 1), (1, 2, 1), (1, 1, 2), (1 + 2 ** 32, 1, 1), (1, 1 + 2 ** 32, 1))]
    q = 1 - int(p * 65536 + 0.5) / 65536
    for i, a in enumerate(masks):
        # five standard deviations of a share of n independent draws
        assert abs(a.double().mean().item() - q) < 5 * math.sqrt(q * (1 - q) / n)
        for b in masks[:i]:
            both = q * q
            assert abs((a & b).double().mean().item() - both) < 5 * math.sqrt(both * (1 - both) / n)


def test_linear_act_and_dropout_draw_the_same_mask(ops):
    torch.manual_seed(2)
    rng = rng_of(11, 12)
    for M, N in ((70, 96), (33, 101)):
        x, w = torch.randn(M, 64, device="cuda").to(BF), torch.randn(N, 64, device="cuda").to(BF)
        a, b = ops.linear_act(x, w, p=0.4, rng=rng, site=3), ops.dropout(ops.linear_act(x, w), 0.4, rng, 3)
        assert torch.equal(a == 0, b == 0) and 0.3 < (a == 0).float().mean() < 0.5


def test_elements_past_the_32nd_bit(ops):
    """A tensor of more than 2^32 elements: groups past 2^29, and a product whose output has them."""
    rows, n = 65537, 65536 + 8
    rng = rng_of(21, 22)
    total = rows * n
    assert total > 2 ** 32 + 2 ** 19
    x = torch.ones(rows, n, device="cuda", dtype=BF)
    tail = [total - 5, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 12345, total - 1]

    def kept(i):
        words = plain_bits(21, 22, 1, i >> 3)
        return (words[(i & 7) >> 1] >> (i & 1) * 16 & 0xFFFF) >= 32768
    y = ops.dropout(x, 0.5, rng, 1).view(-1)
    assert [float(y[i]) for i in tail] == [2.0 * kept(i) for i in tail]
    del x, y
    a, w = torch.ones(rows, 8, device="cuda", dtype=BF), torch.ones(n, 8, device="cuda", dtype=BF)
    y = ops.linear_act(a, w, p=0.5, rng=rng, site=1).view(-1)
    assert [float(y[i]) for i in tail] == [16.0 * kept(i) for i in tail]
    assert abs((y[-1000000:] != 0).float().mean().item() - 0.5) < 0.005


# ------------------------------------------------------------------------------------------------------------ loss
def loss64(x, w, target, ignore=-100):
    """float64 losses per row, logsumexp, probabilities, and a bound on a logit's error."""
    xd, wd = x.double(), w.double()
    counts = target != ignore
    xd = torch.where(counts[:, None], xd, 0.0)
    logits = xd @ wd.T
    delta = acc(x.shape[1]) * (xd.abs() @ wd.abs().T).amax(1)
    lse = torch.logsumexp(logits, 1)
    rows = torch.where(counts, lse - logits.gather(1, target.clamp(0)[:, None])[:, 0], 0.0)
    return rows, lse, logits, delta, counts, xd, wd


def check_loss(ops, x, w, target, reduction, upstream=None):
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = ops.linear_cross_entropy(xl, wl, target, reduction=reduction)
    rows, lse, logits, delta, counts, xd, wd = loss64(x, w, target)
    n = max(1, int(counts.sum()))
    row_err = torch.where(counts, 2 * delta + 2.0 ** -20 * (1 + lse.abs()) + 2.0 ** -23 * rows.abs(), 0.0)
    if reduction == "none":
        within(out.detach(), rows, row_err, "losses")
        g = upstream if upstream is not None else torch.randn(len(rows), device="cuda")
        c = g.double()
    else:
        want = rows.sum() / (n if reduction == "mean" else 1)
        within(out.detach(), want, row_err.sum() / (n if reduction == "mean" else 1) + 2.0 ** -23 * want.abs(), "loss")
        g = torch.tensor(1.0 if upstream is None else upstream, device="cuda")
        c = g.double() / (n if reduction == "mean" else 1)
    c = torch.where(counts, c, 0.0)[:, None]
    dx, dw = torch.autograd.grad(out, (xl, wl), g)
    prob = torch.exp(logits - lse[:, None])
    d = prob.clone()
    d[torch.arange(len(rows), device="cuda"), target.clamp(0)] -= 1
    d_err = (prob * (3 * delta[:, None] + 2.0 ** -19 * (1 + lse.abs()[:, None])) + (U + 2.0 ** -22) * d.abs()) * c.abs()
    d = d * c
    want = d @ wd
    within(dx, want, U * want.abs() + d_err @ wd.abs() + acc(w.shape[0]) * (d.abs() @ wd.abs()), "dx")
    want = d.T @ xd
    within(dw, want, U * want.abs() + d_err.T @ xd.abs() + acc(x.shape[0]) * (d.abs().T @ xd.abs()), "dw")
    assert not dx[~counts].any()
    return out.detach(), dx, dw


LOSS_SIZES = [(1, 1, 8), (1, 1000, 64), (3, 7, 8), (16, 1000, 64), (130, 515, 72), (257, 2050, 136), (77, 30522, 64), (300, 128, 1024), (600, 4096, 200), (2100, 5003, 248)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("T,V,H", LOSS_SIZES)
def test_linear_cross_entropy(ops, T, V, H, reduction):
    torch.manual_seed(T + V)
    x, w = torch.randn(T, H, device="cuda").to(BF), (torch.randn(V, H, device="cuda") * 2 / math.sqrt(H)).to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    check_loss(ops, x, w, target, reduction)
    target[::3] = -100
    out = check_loss(ops, x, w, target, reduction, None if reduction == "none" else -2.5)
    for q in (7, 1):   # the same bits from any CTA count
        ops.set_sm_quota(q)
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        again = ops.linear_cross_entropy(xl, wl, target, reduction=reduction)
        ops.set_sm_quota(0)
        assert torch.equal(again.detach(), out[0])


def test_loss_in_several_pieces_of_the_vocabulary(ops):
    """More rows than one piece's scratch holds: gradients of x add up over the pieces, a ragged last one among them."""
    from orion_b200 import kernels
    T, V, H = 9000, 17003, 64
    assert kernels.lib().ob200_linear_cross_entropy_backward_workspace(T, V, H, 1, 1) < T * V * 2
    torch.manual_seed(1)
    x, w = torch.randn(T, H, device="cuda").to(BF), (torch.randn(V, H, device="cuda") * 0.25).to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    target[5:900] = -100
    _, dx, dw = check_loss(ops, x, w, target, "mean")
    # each gradient alone is the same
    a = ops.linear_cross_entropy(x.requires_grad_(True), w, target)
    assert torch.equal(torch.autograd.grad(a, x)[0], dx)
    b = ops.linear_cross_entropy(x.detach(), w.requires_grad_(True), target)
    assert torch.equal(torch.autograd.grad(b, w)[0], dw)


@pytest.mark.parametrize("T,V,H,counted", [(700, V, H, n) for V, H in ((1000, 64), (5003, 136), (2050, 1024)) for n in (0, 1, 63, 64, 65, 128, 129, 300, 512, 513, 699, 700)] +
                         [(1143, 9000, 768, n) for n in (170, 257)] + [(5000, 24001, 136, n) for n in (0, 40, 600, 3000, 4999)] + [(2100, 20000, 264, 200)])
def test_loss_over_the_rows_that_count(ops, T, V, H, counted):
    """Rows that count are packed for the products: none of them, a block, a tile, one more and one less; whatever the others hold; few of
    many, whose gradient products are cut otherwise; in two pieces of the vocabulary; and the same bits from any CTA count."""
    torch.manual_seed(V + counted)
    x, w = torch.randn(T, H, device="cuda").to(BF), (torch.randn(V, H, device="cuda") * 2 / math.sqrt(H)).to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    out = torch.randperm(T, device="cuda")[counted:]
    target[out] = -100
    junk = x.clone()
    junk[out] = float("nan")

    def run(rows, reduction, g, q):
        ops.set_sm_quota(q)
        xl, wl = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = ops.linear_cross_entropy(xl, wl, target, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (xl, wl), g)
        ops.set_sm_quota(0)
        return loss.detach(), dx, dw

    for reduction, g in (("mean", torch.tensor(1.0, device="cuda")), ("none", torch.randn(T, device="cuda"))):
        want = check_loss(ops, x, w, target, reduction, g if reduction == "none" else 1.0)
        for q in (0, 9, 1):
            for a, b in zip(run(junk, reduction, g, q), want):
                assert torch.equal(a, b)
    # each gradient alone: the sums may be cut otherwise, two roundings of nearly the same number
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(ops.linear_cross_entropy(xl, wl, target, reduction="sum"), (xl, wl))
    alone = (torch.autograd.grad(ops.linear_cross_entropy(xl, w, target, reduction="sum"), xl)[0],
             torch.autograd.grad(ops.linear_cross_entropy(x, wl, target, reduction="sum"), wl)[0])
    for a, b in zip(alone, both):
        assert (a - b).abs().max().item() <= 2.0 ** -7 * b.abs().max().item()


def test_more_rows_than_a_forward_pass_has_under_way(ops):
    T, V, H = 65536 + 130, 200, 16
    torch.manual_seed(2)
    x, w = torch.randn(T, H, device="cuda").to(BF), torch.randn(V, H, device="cuda").to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    rows, lse, _, delta, _, _, _ = loss64(x, w, target)
    out = ops.linear_cross_entropy(x, w, target, reduction="none")
    within(out, rows, 2 * delta + 2.0 ** -20 * (1 + lse.abs()) + 2.0 ** -23 * rows.abs(), "losses")
    within(ops.linear_cross_entropy(x, w, target), rows.mean(), (2 * delta + 2.0 ** -20 * (1 + lse.abs())).mean() + 2.0 ** -23 * rows.mean(), "mean")
    # the second block of rows is packed by itself, the first one empty
    target[:65536 + 7] = -100
    out = ops.linear_cross_entropy(x, w, target, reduction="none")
    assert not out[:65536 + 7].any()
    within(out[65536 + 7:], rows[65536 + 7:], (2 * delta + 2.0 ** -20 * (1 + lse.abs()) + 2.0 ** -23 * rows.abs())[65536 + 7:], "losses")
    target[:] = -100
    assert ops.linear_cross_entropy(x, w, target).item() == 0


def test_rows_that_do_not_count_and_labels_that_do_not_exist(ops):
    torch.manual_seed(3)
    T, V, H = 40, 300, 64
    x, w = torch.randn(T, H, device="cuda").to(BF), torch.randn(V, H, device="cuda").to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    target[::2] = -100
    clean = check_loss(ops, x, w, target, "mean")
    for junk in (float("nan"), float("inf"), -float("inf"), 3e38):
        dirty = x.clone()
        dirty[::2] = junk
        xl, wl = dirty.requires_grad_(True), w.clone().requires_grad_(True)
        loss = ops.linear_cross_entropy(xl, wl, target)
        dx, dw = torch.autograd.grad(loss, (xl, wl))
        assert torch.equal(loss.detach(), clean[0]) and torch.equal(dx, clean[1]) and torch.equal(dw, clean[2])
    # no row counts: no loss, no gradient, nothing that is not a number
    none = torch.full((T,), -100, device="cuda")
    for reduction in ("mean", "sum", "none"):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = ops.linear_cross_entropy(xl, wl, none, reduction=reduction)
        dx, dw = torch.autograd.grad(loss.sum(), (xl, wl))
        assert not loss.any() and not dx.any() and not dw.any()
    # any index may be the one that is ignored, one of the vocabulary among them
    few = torch.randint(0, 3, (T,), device="cuda")
    a, b = (ops.linear_cross_entropy(x, w, t, ignore_index=i) for t, i in ((few, 1), (torch.where(few == 1, -100, few), -100)))
    assert torch.equal(a, b)
    # a label outside the vocabulary shows: its loss and the gradients it would have reached are not numbers
    for label in (V, -1, V + 2 ** 32, 2 ** 62):
        bad = target.clone()
        bad[1] = label
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        rows = ops.linear_cross_entropy(xl, wl, bad, reduction="none")
        assert torch.equal(rows.isnan().nonzero().flatten(), torch.tensor([1], device="cuda"))
        dx, dw = torch.autograd.grad(rows.sum(), (xl, wl))
        assert dx[1].isnan().all() and not dx[0].isnan().any() and not dx[2:].isnan().any() and dw.isnan().all()


def test_logits_of_any_size(ops):
    """Logits of +-10^4 (a softmax that overflows without its maximum), equal logits, and infinite ones."""
    T, V, H = 20, 777, 8
    torch.manual_seed(5)
    x, w = (torch.randn(T, H, device="cuda") * 100).to(BF), (torch.randn(V, H, device="cuda") * 100).to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    check_loss(ops, x, w, target, "none")
    same = ops.linear_cross_entropy(torch.zeros_like(x), w, target, reduction="none")
    within(same, torch.full((T,), math.log(V), dtype=torch.float64, device="cuda"), torch.tensor(2.0 ** -20 * 8, device="cuda"), "equal logits")
    # one word at minus infinity weighs nothing; the row whose label it is has an infinite loss
    one, vocab = torch.ones(T, H, device="cuda").to(BF), torch.randn(V, H, device="cuda").to(BF)
    low = vocab.clone()
    low[5] = -float("inf")
    target[:] = 9
    target[3] = 5
    got = ops.linear_cross_entropy(one, low, target, reduction="none")
    want = ops.linear_cross_entropy(one, torch.cat([vocab[:5], vocab[6:]]), torch.where(target == 9, 8, 0), reduction="none")
    assert got[3].item() == float("inf")
    within(got[4:], want[4:].double(), 2.0 ** -19 * (1 + want[4:].double().abs()), "without the word")
    # not a number stays one
    low[5] = float("nan")
    assert ops.linear_cross_entropy(one, low, target, reduction="none").isnan().all()
    assert ops.linear_cross_entropy(one, torch.full_like(vocab, float("nan")), target, reduction="none").isnan().all()


def test_loss_layouts_and_empty_batches(ops):
    torch.manual_seed(6)
    big, w = torch.randn(6, 11, 80, device="cuda").to(BF), torch.randn(99, 144, device="cuda").to(BF)
    for x, weight in ((big[:, :, :64], w[:, :64]), (big[:, 1:, 3:67].transpose(0, 1), w[:, 9:73]), (big[:, ::2, 8:72], w[:, 80:].T.contiguous().T)):
        target = torch.randint(0, 99, x.shape[:-1][::-1], device="cuda").T
        xl, wl = x.detach().requires_grad_(True), weight.detach().requires_grad_(True)
        rows = ops.linear_cross_entropy(xl, wl, target, reduction="none")
        assert rows.shape == target.shape
        g = torch.randn(rows.shape[::-1], device="cuda").T
        xc, wc = x.reshape(-1, 64).contiguous().requires_grad_(True), weight.contiguous().requires_grad_(True)
        flat = ops.linear_cross_entropy(xc, wc, target.reshape(-1), reduction="none")
        assert torch.equal(rows.flatten(), flat)
        for a, b in zip(torch.autograd.grad(rows, (xl, wl), g), torch.autograd.grad(flat, (xc, wc), g.reshape(-1))):
            assert torch.equal(a.flatten(), b.flatten())
    none, wl = torch.empty(0, 64, device="cuda", dtype=BF, requires_grad=True), w[:, :64].detach().requires_grad_(True)
    for reduction in ("mean", "sum", "none"):
        loss = ops.linear_cross_entropy(none, wl, torch.empty(0, dtype=torch.int64, device="cuda"), reduction=reduction)
        assert not loss.any()
        dx, dw = torch.autograd.grad(loss.sum(), (none, wl))
        assert dx.shape == (0, 64) and dw.shape == wl.shape and not dw.any()


def test_loss_gradient_is_the_difference_quotient(ops):
    """L(w + h d) - L(w - h d) over 2 h along d: off by at most h^2 / 6 of the third cumulant of the logits' change, which is at most the
    cube of its range.  w, d and h have few bits, so that w +- h d are exact."""
    torch.manual_seed(7)
    T, V, H, h = 50, 333, 64, 1 / 32
    x = (torch.randint(-4, 5, (T, H), device="cuda") / 8).to(BF)
    w, d = (torch.randint(-8, 9, (V, H), device="cuda") / 16).to(BF), torch.randint(-1, 2, (V, H), device="cuda").to(BF) / 4
    target = torch.randint(0, V, (T,), device="cuda")
    wl = w.clone().requires_grad_(True)
    grad, = torch.autograd.grad(ops.linear_cross_entropy(x, wl, target), wl)
    up, down = (ops.linear_cross_entropy(x, w + s * h * d, target).double() for s in (1, -1))
    along = x.double() @ d.double().T
    spread = along.amax(1) - along.amin(1)
    delta = loss64(x, w, target)[3].max()
    bound = (spread ** 3).mean() * h * h / 6 + (2 * delta + 2.0 ** -20 * 8) / h + (3 * U * grad.double().abs() * d.double().abs()).sum()
    assert abs((up - down) / (2 * h) - (grad.double() * d.double()).sum()) <= bound


# ------------------------------------------------------------------------------------------------------------ streams, graphs, users
def test_another_stream_and_two_calls_at_once(ops):
    torch.manual_seed(8)
    x, w, b, r = make(300, 256, 2048, True, BF, 1)
    rng = rng_of(1, 1)
    target = torch.randint(0, 256, (300,), device="cuda")
    want = ops.linear_act(x, w, b, r, "gelu", 0.1, rng, 1)
    want_loss = ops.linear_cross_entropy(x, w, target)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.linear_act(x, w, b, r, "gelu", 0.1, rng, 1), ops.linear_cross_entropy(x, w, target)))
    torch.cuda.synchronize()
    for a, l in got[0] + got[1]:
        assert torch.equal(a, want) and torch.equal(l, want_loss)


def test_saved_state_that_has_changed_is_noticed(ops):
    x, w, _, _ = make(8, 16, 64, False, None, 1)
    rng = rng_of(1, 1)
    for run in (lambda: ops.linear_act(x.requires_grad_(True), w, p=0.5, rng=rng), lambda: ops.dropout(x.requires_grad_(True), 0.5, rng)):
        y = run()
        rng[1] += 1   # the step moves on before the backward pass has drawn its mask again
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_second_derivatives_are_refused(ops):
    x, w, _, _ = make(8, 16, 64, False, None, 1)
    target = torch.zeros(8, dtype=torch.int64, device="cuda")
    for run in (lambda a: ops.linear_act(a, w, act="gelu"), lambda a: ops.dropout(a, 0.5, rng_of(1, 1)), lambda a: ops.linear_cross_entropy(a, w, target)):
        a = x.clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="twice"):
            g, = torch.autograd.grad(run(a).float().sum(), a, create_graph=True)
            torch.autograd.grad(g.float().sum(), a)


def step_of(ops, m, ids, target, rng, p):
    """A decoder block's feed-forward half, training: embedding dropout, GELU layer, residual branch with dropout, norm, loss."""
    x = ops.dropout(m["emb"][ids], p, rng, 0)
    hid = ops.linear_act(x, m["w1"], m["b1"], None, "gelu")
    x = ops.linear_act(hid, m["w2"], m["b2"], x, "none", p, rng, 1)
    x = ops.layernorm_train(x, m["g"], m["s"], 1e-5)
    return ops.linear_cross_entropy(x, m["head"], target)


def model(seed, V=515, h=128, ffn=264):
    torch.manual_seed(seed)
    m = {"emb": torch.randn(V, h), "w1": torch.randn(ffn, h) / math.sqrt(h), "b1": torch.randn(ffn) * 0.1, "w2": torch.randn(h, ffn) / math.sqrt(ffn),
         "b2": torch.randn(h) * 0.1, "g": torch.rand(h) + 0.5, "s": torch.randn(h) * 0.1, "head": torch.randn(V, h) / math.sqrt(h)}
    return {k: v.to("cuda", BF).requires_grad_(True) for k, v in m.items()}


def test_the_operators_together(ops):
    """One step of embedding, feed-forward, dropout, norm and loss against float64 with the same masks: 2e-2 of each tensor's largest
    entry, the bound of the framework's other whole-layer tests (five bfloat16 roundings of activations on the way, 2^-8 each)."""
    m, rng, p = model(0), rng_of(77, 5), 0.1
    B, S, V = 3, 50, 515
    ids, target = torch.randint(0, V, (B, S), device="cuda"), torch.randint(0, V, (B, S), device="cuda")
    target[:, 40:] = -100
    before = ops.fallbacks()
    loss = step_of(ops, m, ids, target, rng, p)
    grads = torch.autograd.grad(loss, list(m.values()))
    assert ops.fallbacks() == before
    d = {k: v.detach().double().requires_grad_(True) for k, v in m.items()}
    masks = []
    for site in (0, 1):
        keep, f = keep_mask(B * S * 128, p, rng, site)
        masks.append(keep.view(B, S, 128).double() * f)
    x = d["emb"][ids] * masks[0]
    x = x + (torch.nn.functional.gelu(x @ d["w1"].T + d["b1"]) @ d["w2"].T + d["b2"]) * masks[1]
    x = torch.nn.functional.layer_norm(x, (128,), d["g"], d["s"], 1e-5)
    want = torch.nn.functional.cross_entropy((x @ d["head"].T).flatten(0, 1), target.flatten())
    assert abs(loss.item() - want.item()) < 2e-2 * want.item()
    for (name, _), g, gd in zip(m.items(), grads, torch.autograd.grad(want, list(d.values()))):
        assert (g.double() - gd).abs().max() <= 2e-2 * gd.abs().max(), name


def test_captured_training_steps_replayed_side_by_side(ops):
    """Two captured steps on two streams, replayed at once and over again: each as the eager step of its inputs and its step count, which
    moves on inside the graph."""
    V, B, S, p = 515, 2, 130, 0.1
    graphs, want = [], []
    for k in range(2):
        m, rng = model(k), rng_of(7 + k, 100)
        ids, target = torch.randint(0, V, (B, S), device="cuda"), torch.randint(0, V, (B, S), device="cuda")
        expected = []
        for step in range(3):
            loss = step_of(ops, m, ids, target, rng_of(7 + k, 100 + step), p)
            expected.append([loss.detach()] + list(torch.autograd.grad(loss, list(m.values()))))
            del loss
        want.append(expected)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                torch.autograd.grad(step_of(ops, m, ids, target, rng, p), list(m.values()))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            loss = step_of(ops, m, ids, target, rng, p)
            out = [loss.detach()] + list(torch.autograd.grad(loss, list(m.values())))
            rng[1:] += 1
        graphs.append((g, s, out, m, rng, ids, target))
    torch.cuda.synchronize()
    for step in range(3):
        for g, s, *_ in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, out, m, *_), expected in zip(graphs, want):
            for name, a, b in zip(["loss"] + list(m), out, expected[step]):
                if name == "emb":   # the table's gradient is the stock index kernel's, whose atomics have no order
                    assert (a.double() - b.double()).abs().max() <= 4 * U * b.double().abs().max()
                else:
                    assert torch.equal(a, b), (name, step)


def test_inference_mode_and_no_grad(ops):
    x, w, b, r = make(40, 64, 128, True, BF, 3)
    target = torch.randint(0, 64, (40,), device="cuda")
    rng = rng_of(1, 2)
    a = (ops.linear_act(x, w, b, r, "gelu", 0.2, rng), ops.dropout(x, 0.2, rng), ops.linear_cross_entropy(x, w, target))
    for mode in (torch.no_grad(), torch.inference_mode()):
        with mode:
            y = (ops.linear_act(x.requires_grad_(False), w, b, r, "gelu", 0.2, rng), ops.dropout(x, 0.2, rng), ops.linear_cross_entropy(x, w, target))
            assert all(torch.equal(p, q) and not q.requires_grad for p, q in zip(a, y))


def test_through_the_c_abi(built):
    """The ctypes binding: the same results as the operators, outputs where the caller wants them."""
    from orion_b200 import kernels as K, torch_ops
    ops = torch_ops.load()
    x, w, b, r = make(300, 250, 2056, True, torch.float32, 5)
    rng, target = rng_of(3, 4), torch.randint(0, 250, (300,), device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dy = torch.randn(300, 250, device="cuda").to(BF)
    y = ops.linear_act(x, w, b, r, "gelu", 0.1, rng, 6)
    want = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        mine, slope = K.linear_act(x, w, b, r, "gelu", 0.1, rng, 6, want_slope=True, num_ctas=40)
        assert torch.equal(mine, y)
        for g, h in zip(K.linear_act_backward(dy, slope, x, w, torch.float32, "gelu", 0.1, rng, 6, num_ctas=33), want):
            assert torch.equal(g, h)
        assert torch.equal(K.dropout(r, 0.3, rng, 1, num_ctas=3), ops.dropout(r, 0.3, rng, 1))
    loss = ops.linear_cross_entropy(x, w, target)
    want = torch.autograd.grad(loss, (x, w))
    with torch.no_grad():
        total, rows, lse, count = K.linear_cross_entropy(x, w, target, num_ctas=50)
        assert torch.equal(total, loss) and count.item() == 300
        for g, h in zip(K.linear_cross_entropy_backward(x, w, target, lse, torch.ones((), device="cuda"), count, num_ctas=21), want):
            assert torch.equal(g, h)


@pytest.mark.parametrize("T,V,H,counted", [(1143, 9000, 768, 171), (1143, 9000, 768, 1143), (700, 5003, 136, 3), (5000, 24001, 136, 40), (300, 128, 1024, 100), (40, 515, 64, 20)])
def test_calls_stay_inside_their_scratch_and_outputs(built, T, V, H, counted):
    """Guard words behind the scratch and behind every output of the loss and of the linear layer stay as they were."""
    from orion_b200 import kernels as K
    L, guard = K.lib(), 1 << 20
    torch.manual_seed(T + counted)
    x, w = torch.randn(T, H, device="cuda").to(BF), torch.randn(V, H, device="cuda").to(BF)
    target = torch.randint(0, V, (T,), device="cuda")
    target[torch.randperm(T, device="cuda")[counted:]] = -100
    spaces = []

    def space(n):
        t = torch.full((n + guard,), 0xA5, device="cuda", dtype=torch.uint8)
        spaces.append((t, n))
        return t
    loss, lse, total, count, dx, dw = space(T * 4), space(T * 4), space(4), space(4), space(T * H * 2), space(V * H * 2)
    one = torch.ones((), device="cuda")
    n = L.ob200_linear_cross_entropy_workspace(T, V, H)
    assert L.ob200_linear_cross_entropy_forward(*(K._ptr(t) for t in (x, w, target, loss, lse, total, count)), T, V, H, H, H, -100, 1, K._ptr(space(n)), n,
                                                K.sm_count(), K._stream()) == 0
    n = L.ob200_linear_cross_entropy_backward_workspace(T, V, H, 1, 1)
    assert L.ob200_linear_cross_entropy_backward(*(K._ptr(t) for t in (x, w, target, lse, one)), 0, K._ptr(count), K._ptr(dx), K._ptr(dw), T, V, H, H, H,
                                                 -100, K._ptr(space(n)), n, K.sm_count(), K._stream()) == 0
    N = 515   # a linear layer of the same input
    wl, bias, dy, rng = torch.randn(N, H, device="cuda").to(BF), torch.randn(N, device="cuda").to(BF), torch.randn(T, N, device="cuda").to(BF), rng_of(1, 2)
    y, slope, dxl, dwl, db = space(T * N * 2), space(T * 520 * 2), space(T * H * 2), space(N * H * 2), space(N * 2)
    n = L.ob200_linear_act_workspace(T, N, H)
    assert L.ob200_linear_act_bf16(*(K._ptr(t) for t in (x, wl, y, slope, bias)), 0, None, 2, 0.1, K._ptr(rng), 0, T, N, H, H, H, 520, K._ptr(space(n)), n,
                                   K.sm_count(), K._stream()) == 0
    n = L.ob200_linear_act_backward_workspace(T, N, H, 2, 0.1, 1, 1, 1)
    assert L.ob200_linear_act_backward_bf16(*(K._ptr(t) for t in (dy, slope, x, wl, dxl, dwl, db)), 0, 2, 0.1, K._ptr(rng), 0, T, N, H, H, H, 520,
                                            K._ptr(space(n)), n, K.sm_count(), K._stream()) == 0
    for t, n in spaces:
        assert (t[n:] == 0xA5).all(), n


def test_gradients_over_no_rows_are_zeros(built):
    from orion_b200 import kernels as K
    L = K.lib()
    x, w, dy = torch.empty(0, 64, device="cuda", dtype=BF), torch.ones(40, 64, device="cuda", dtype=BF), torch.empty(0, 40, device="cuda", dtype=BF)
    dw, db = torch.ones(40, 64, device="cuda", dtype=BF), torch.ones(40, device="cuda")
    assert L.ob200_linear_act_backward_bf16(K._ptr(dy), None, K._ptr(x), K._ptr(w), None, K._ptr(dw), K._ptr(db), 1, 0, 0.0, None, 0, 0, 40, 64, 64, 64, 0,
                                            None, 0, K.sm_count(), K._stream()) == 0
    assert not dw.any() and not db.any()
    dx = torch.ones(5, 64, device="cuda", dtype=BF)
    assert L.ob200_linear_act_backward_bf16(K._ptr(dy), None, K._ptr(x), K._ptr(w), K._ptr(dx), None, None, 1, 0, 0.0, None, 0, 5, 0, 64, 64, 64, 0,
                                            None, 0, K.sm_count(), K._stream()) == 0
    assert not dx.any()


def test_a_captured_loss_counts_its_rows_anew_at_each_replay(ops):
    """How many rows count is read on the device: a graph captured with one number of them is right for every other."""
    T, V, H = 900, 5003, 264
    torch.manual_seed(4)
    x, w = torch.randn(T, H, device="cuda").to(BF).requires_grad_(True), (torch.randn(V, H, device="cuda") / 8).to(BF).requires_grad_(True)
    labels, target = torch.randint(0, V, (T,), device="cuda"), torch.empty(T, device="cuda", dtype=torch.long)
    target.copy_(labels)
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
    for counted in (900, 1, 0, 257, 256, 899, 64, 900):
        target.copy_(labels)
        target[torch.randperm(T, device="cuda")[counted:]] = -100
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.linear_cross_entropy(x, w, target)
        want = [eager.detach()] + list(torch.autograd.grad(eager, (x, w)))
        for a, b in zip(out, want):
            assert torch.equal(a, b), counted
        del eager


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("M,N", [(2200, 2040), (264, 1000), (1040, 512)])
def test_gemm_tiles_whose_lower_warps_are_past_the_edge(built, M, N, out_dtype):
    """A warp with no rows in the last row of tiles must not run over the slab that its store of the tile before still reads: the same
    bits time after time, from one CTA (all tiles in a row) and from all."""
    from orion_b200 import kernels as K
    torch.manual_seed(M)
    a, b = torch.randn(M, 136, device="cuda").to(BF), torch.randn(N, 136, device="cuda").to(BF)
    want = K.gemm_bf16(a, b, out_dtype=out_dtype)
    for _ in range(60):
        for ctas in (1, 7):
            assert torch.equal(K.gemm_bf16(a, b, out_dtype=out_dtype, num_ctas=ctas), want)
