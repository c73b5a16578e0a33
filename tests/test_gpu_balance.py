"""GPU: the router's balance loss, its counts and its gradient, against
float64 on the CPU and against differences."""
import pytest
import torch

import mx_reference as R
from conftest import pkg

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _inputs(T, E, K, S, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)
    ids = (x.topk(K, 1).indices if T else torch.zeros(0, K)).int()
    cut = torch.randint(0, T + 1, (S - 1,), generator=g).sort().values
    off = torch.cat((torch.zeros(1), cut, torch.full((1,), float(T)))).int()
    return x.to(dtype), ids, off, torch.rand(S, generator=g) + 0.5


def _check(x, ids, off, grad, score, coeff=0.3):
    xd = x.to(DEV).requires_grad_(True)
    offd = None if off is None else off.to(DEV)
    loss, counts = pkg().balance_loss(xd, ids.to(DEV), offd, coeff, score)
    dx, = torch.autograd.grad(loss, xd, grad.to(DEV))
    want, n, back = R.balance(x.float(), ids, off, coeff, score)
    assert counts.dtype == torch.int32 and torch.equal(counts.cpu().long(), n)
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    # a score: exp (2 steps), add, divide; the row's sum (log2 E + E / 32 adds), the reciprocal and product; a
    # column's sum of a run's tokens; each at most 2^-24 of the value (every term is positive): under 128 of them
    # and one for each 64 tokens of a run
    T, E = x.shape
    rel = (128 + E / 32 + T / 64) * 2.0 ** -24
    torch.testing.assert_close(loss.cpu().double(), want, rtol=rel, atol=0)
    # d = g c / T_s p_j (f_j - sum f p) (..): the difference cancels, so the error is relative to its two terms
    assert dx.dtype == x.dtype and dx.shape == x.shape
    off_l = [0, T] if off is None else off.tolist()
    ref = back(grad)
    tol = torch.zeros(T, E, dtype=torch.float64)
    for s, (lo, hi) in enumerate(zip(off_l[:-1], off_l[1:])):
        if hi > lo:
            r = x[lo:hi].double()
            p = torch.softmax(r, 1) if score == "softmax" else r.sigmoid() / r.sigmoid().sum(1, keepdim=True)
            f = n[s].double() * E / (ids.shape[1] * (hi - lo))
            tol[lo:hi] = rel * grad[s].double() * coeff / (hi - lo) * p * (f + (p * f).sum(1, keepdim=True))
    tol += torch.finfo(x.dtype).eps / 2 * 1.01 * ref.abs() + torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    assert ((dx.cpu().double() - ref).abs() <= tol).all()
    return loss, dx


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,K,S,dtype", [
    (1, 256, 8, 1, "fp32"), (7, 8, 2, 3, "fp32"), (1000, 256, 8, 5, "fp32"), (1000, 256, 8, 40, "bf16"),
    (333, 60, 4, 7, "fp16"), (129, 1, 1, 2, "fp32"), (50, 1024, 8, 3, "fp32"), (77, 513, 6, 4, "bf16"),
    (9000, 64, 6, 2, "fp32"), (5, 160, 6, 64, "fp32")])
def test_balance_loss(gpu_available, score, T, E, K, S, dtype):
    _check(*_inputs(T, E, K, S, R.DTYPES[dtype], T + E + S), score)


def test_one_sequence_without_offsets_and_strided_logits(gpu_available):
    x, ids, _, grad = _inputs(100, 96, 4, 1, torch.float32, 3)
    _check(x, ids, None, grad, "sigmoid")
    wide = torch.zeros(100, 131)
    wide[:, 17:113] = x
    view = wide.to(DEV)[:, 17:113].requires_grad_(True)
    loss, _ = pkg().balance_loss(view, ids.to(DEV), None, 0.3)
    want, _, back = R.balance(x, ids, None, 0.3, "sigmoid")
    torch.testing.assert_close(loss.detach().cpu().double(), want, rtol=2.0 ** -16, atol=0)
    dx, = torch.autograd.grad(loss.sum(), view)
    assert dx.shape == x.shape
    torch.testing.assert_close(dx.cpu().double(), back(torch.ones(1)), rtol=1e-3, atol=1e-9)


def test_ids_outside_repeated_and_tokens_of_no_sequence(gpu_available):
    x, ids, _, _ = _inputs(64, 32, 4, 1, torch.float32, 4)
    ids[3] = torch.tensor([-1, 32, 1 << 30, -(1 << 31)])
    ids[4] = 7
    off = torch.tensor([5, 20, 20, 50], dtype=torch.int32)
    _, dx = _check(x, ids, off, torch.tensor([1.0, 2.0, 0.5]), "softmax")
    assert (dx[:5] == 0).all() and (dx[50:] == 0).all() and (dx[5:50] != 0).any()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_masked_logits(gpu_available, score):
    """-inf in places, a row of them, the type's lowest value, a NaN row."""
    x, ids, off, grad = _inputs(40, 64, 4, 2, torch.float32, 5)
    x[1, :60] = -torch.inf
    x[2] = -torch.inf
    x[3, 5] = torch.finfo(torch.float32).min
    xd = x.to(DEV).requires_grad_(True)
    loss, counts = pkg().balance_loss(xd, ids.to(DEV), off.to(DEV), 1.0, score)
    dx, = torch.autograd.grad(loss, xd, grad.to(DEV))
    assert loss.isfinite().all() and dx.isfinite().all() and (dx[2] == 0).all() and (dx[1, :60] == 0).all()
    keep = torch.ones(40, dtype=torch.bool)
    keep[2] = False
    # without the empty row's terms: its p is 0 and its ids still count
    y = x.double()[keep]
    p = torch.zeros(40, 64, dtype=torch.float64)
    p[keep] = torch.softmax(y, 1) if score == "softmax" else y.sigmoid() / y.sigmoid().sum(1, keepdim=True)
    for s in range(2):
        lo, hi = int(off[s]), int(off[s + 1])
        if hi > lo:
            f = counts[s].cpu().double() * 64 / (4 * (hi - lo))
            want = (f * p[lo:hi].sum(0) / (hi - lo)).sum()
            torch.testing.assert_close(loss[s].detach().cpu().double(), want, rtol=2.0 ** -16, atol=0)
    x[0, 0] = torch.nan
    loss, _ = pkg().balance_loss(x.to(DEV), ids.to(DEV), torch.tensor([0, 1, 40], dtype=torch.int32, device=DEV), 1.0, score)
    assert loss[0].isnan() and loss[1].isfinite()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_gradient_against_differences(gpu_available, score):
    """Central differences of the float64 loss with the kernel's gradient: the
    step 1e-4 leaves an error of 1e-8 of the third derivative's size."""
    x, ids, off, grad = _inputs(6, 16, 2, 2, torch.float32, 6)
    xd = x.to(DEV).requires_grad_(True)
    loss, _ = pkg().balance_loss(xd, ids.to(DEV), off.to(DEV), 1.0, score)
    dx, = torch.autograd.grad(loss, xd, grad.to(DEV))
    for t, j in ((0, 3), (2, 15), (5, 0), (4, 8)):
        d = []
        for h in (-1e-4, 1e-4):
            y = x.double()
            y[t, j] += h
            d.append((R.balance(y, ids, off, 1.0, score)[0] * grad.double()).sum())
        assert abs(float((d[1] - d[0]) / 2e-4) - float(dx[t, j])) < 2e-6


def test_empty_repeat_graph_and_backward_twice(gpu_available):
    m = pkg()
    e = torch.empty(0, 16, device=DEV, requires_grad=True)
    loss, counts = m.balance_loss(e, torch.empty(0, 2, dtype=torch.int32, device=DEV),
                                  torch.zeros(3, dtype=torch.int32, device=DEV))
    assert (loss == 0).all() and (counts == 0).all()
    g, = torch.autograd.grad(loss.sum(), e)
    assert g.shape == (0, 16)
    x, ids, off, grad = _inputs(500, 256, 8, 6, torch.float32, 8)
    xd, idd, offd, gd = x.to(DEV).requires_grad_(True), ids.to(DEV), off.to(DEV), grad.to(DEV)
    loss, _ = m.balance_loss(xd, idd, offd)
    a, = torch.autograd.grad(loss, xd, gd, retain_graph=True)
    b, = torch.autograd.grad(loss, xd, gd)
    assert torch.equal(a, b)
    loss2, _ = m.balance_loss(xd.detach(), idd, offd)
    assert torch.equal(loss, loss2) and not loss2.requires_grad
    graph = torch.cuda.CUDAGraph()
    xs = xd.detach().clone()
    with torch.cuda.graph(graph):
        lg, cg = m.balance_loss(xs, idd, offd)
    xs.copy_(xd.detach() * 0.5)
    graph.replay()
    torch.cuda.synchronize()
    want, n, _ = R.balance(x * 0.5, ids, off, 1e-4, "sigmoid")
    torch.testing.assert_close(lg.cpu().double(), want, rtol=2.0 ** -16, atol=0)
    assert torch.equal(cg.cpu().long(), n)


def test_forward_and_backward_in_a_graph(gpu_available):
    """The whole step captured, replayed on new logits; a call on another
    stream meanwhile, with a workspace of its own."""
    m = pkg()
    x, ids, off, grad = _inputs(700, 256, 8, 5, torch.float32, 12)
    idd, offd, gd = ids.to(DEV), off.to(DEV), grad.to(DEV)
    xs = x.to(DEV).requires_grad_(True)

    def step():
        loss, _ = m.balance_loss(xs, idd, offd, 0.5, "softmax")
        return loss, torch.autograd.grad(loss, xs, gd)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dx = step()
    y = (0.3 * x).to(DEV)
    with torch.no_grad():
        xs.copy_(y)
    torch.cuda.synchronize()
    graph.replay()
    with torch.cuda.stream(side):
        other = [m.balance_loss(y, idd, offd, 0.5, "softmax")[0] for _ in range(20)]
    torch.cuda.synchronize()
    want, _, back = R.balance(0.3 * x, ids, off, 0.5, "softmax")
    torch.testing.assert_close(loss.detach().cpu().double(), want, rtol=2.0 ** -16, atol=0)
    assert all(torch.equal(o, loss) for o in other)
    ref = back(grad)
    assert (dx.cpu().double() - ref).norm() <= 2.0 ** -16 * ref.norm()


def test_second_derivative_is_refused(gpu_available):
    x, ids, off, _ = _inputs(8, 16, 2, 1, torch.float32, 9)
    xd = x.to(DEV).requires_grad_(True)
    loss, _ = pkg().balance_loss(xd, ids.to(DEV), off.to(DEV))
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(loss.sum(), xd, create_graph=True)


def test_training_step_with_the_router(gpu_available):
    """route's ids, the loss added to another one, gradients through a weight
    matrix; the bias update's counts."""
    m = pkg()
    g = torch.Generator().manual_seed(10)
    h, w = torch.randn(96, 64, generator=g).to(DEV), (0.2 * torch.randn(256, 64, generator=g)).to(DEV).requires_grad_(True)
    bias = torch.zeros(256, dtype=torch.bfloat16, device=DEV)
    logits = h @ w.t()
    ids, _, n = m.route(logits.detach(), bias, 0, 256, 2.5)
    off = torch.tensor([0, 40, 96], dtype=torch.int32, device=DEV)
    loss, counts = m.balance_loss(logits, ids, off, 0.1)
    assert torch.equal(counts.sum(0, dtype=torch.int32), n)
    (loss.sum() + logits.square().mean()).backward()
    wd = w.detach().double().cpu().requires_grad_(True)
    lg = h.double().cpu() @ wd.t()
    want, _, back = R.balance(lg, ids.cpu(), off.cpu(), 0.1, "sigmoid")
    lg.backward(back(torch.ones(2)) + 2 * lg.detach() / lg.numel())
    # float32 products over 64 columns and 96 rows: 2^-24 (64 + 96) of the sum of magnitudes, a few of the result's size
    assert ((w.grad.cpu().double() - wd.grad).norm() / wd.grad.norm()) < 160 * 2.0 ** -24 * 8


def test_refusals(gpu_available):
    m = pkg()
    x = torch.zeros(8, 16, device=DEV)
    ids = torch.zeros(8, 2, dtype=torch.int32, device=DEV)
    for call in (lambda: m.balance_loss(x, ids.long()), lambda: m.balance_loss(x, ids[:4]), lambda: m.balance_loss(x.int(), ids),
                 lambda: m.balance_loss(x.t(), ids), lambda: m.balance_loss(x[0], ids), lambda: m.balance_loss(x, ids, score_func="relu"),
                 lambda: m.balance_loss(x, ids, torch.zeros(3, device=DEV)), lambda: m.balance_loss(x, ids, torch.zeros(3, dtype=torch.int32)),
                 lambda: m.balance_loss(torch.zeros(8, 1025, device=DEV), ids),
                 lambda: m.balance_loss(x, torch.zeros(8, 17, dtype=torch.int32, device=DEV)),
                 lambda: m.balance_loss(x, ids, torch.zeros(1, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            call()


def _formula(x, ids, off, grad, score, coeff):
    """The gradient from its formula in float64, and the sum of its two terms'
    sizes. The sigmoid's complement is sigmoid(-l), which no difference cancels."""
    x = x.double()
    (T, E), K = x.shape, ids.shape[1]
    ref, size = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
    for s, (lo, hi) in enumerate(zip(off[:-1].tolist(), off[1:].tolist())):
        if hi <= lo:
            continue
        r = x[lo:hi]
        p = torch.softmax(r, 1) if score == "softmax" else r.sigmoid() / r.sigmoid().sum(1, keepdim=True)
        f = torch.bincount(ids[lo:hi].flatten().long(), minlength=E).double() * E / (K * (hi - lo))
        unit = grad[s].double() * coeff / (hi - lo) * p * (1.0 if score == "softmax" else (-r).sigmoid())
        mean = (p * f).sum(1, keepdim=True)
        ref[lo:hi], size[lo:hi] = unit * (f - mean), unit * (f + mean)
    return ref, size


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("low,high", [(8, 16), (10, 40), (17, 30), (-40, 40), (-80, -20)])
@pytest.mark.parametrize("T,E,K,S", [(40, 16, 2, 3), (33, 60, 4, 2), (70, 256, 8, 4), (20, 1024, 8, 2), (12, 513, 6, 2)])
def test_gradient_of_large_logits(gpu_available, T, E, K, S, low, high, dtype):
    """The sigmoid's factor 1 - sigmoid(l) is e^-16 and less here: the error
    stays relative to the gradient's own terms, this factor included."""
    _, ids, off, grad = _inputs(T, E, K, S, torch.float32, T + E)
    x = (low + (high - low) * torch.rand(T, E, generator=torch.Generator().manual_seed(E))).to(R.DTYPES[dtype])
    xd = x.to(DEV).requires_grad_(True)
    loss, _ = pkg().balance_loss(xd, ids.to(DEV), off.to(DEV), 0.3)
    dx, = torch.autograd.grad(loss, xd, grad.to(DEV))
    ref, size = _formula(x, ids, off, grad, "sigmoid", 0.3)
    # as in _check, and for the factor an exponential, a sum, a quotient and two products: 16 half-steps more
    rel = (144 + E / 32 + T / 64) * 2.0 ** -24
    tol = rel * size + torch.finfo(x.dtype).eps / 2 * 1.01 * ref.abs() + torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    assert ((dx.cpu().double() - ref).abs() <= tol).all()


def test_gradient_of_saturated_rows_against_differences(gpu_available):
    """Rows whose float32 sigmoids are all 1: differences of the loss in
    float64, p_j = (1 - c_j) / sum (1 - c) with c = sigmoid(-l)."""
    T, E = 4, 8
    g = torch.Generator().manual_seed(3)
    x = 12 + 8 * torch.rand(T, E, generator=g)
    x[1] += 6
    ids = torch.tensor([[0, 1], [2, 0], [0, 3], [1, 0]], dtype=torch.int32)
    xd = x.to(DEV).requires_grad_(True)
    loss, _ = pkg().balance_loss(xd, ids.to(DEV), None, 1.0)
    dx, = torch.autograd.grad(loss.sum(), xd)
    f = torch.bincount(ids.flatten().long(), minlength=E).double() * E / (2 * T)

    def change(t, j, d):
        """loss(l_tj + d) - loss(l_tj) without a difference of nearly equal numbers: the change of a_j is
        D = c (1 - e^-d) / (1 + e^(-l-d)), and that of sum_i f_i p_i is D (f_j - mean) / (sum + D)."""
        a = x[t].double().sigmoid()
        c = (-x[t, j].double()).sigmoid()
        dj = -c * torch.expm1(torch.tensor(-d, dtype=torch.float64)) / (1 + torch.exp(-x[t, j].double() - d))
        mean = (f * a).sum() / a.sum()
        return dj * (f[j] - mean) / (a.sum() + dj) / T

    for t in range(T):
        for j in range(E):
            # the gradient is u (f_j - mean), u = c / (T sum): its error is (144 + ..) 2^-24 < 2^-16 of u (f_j + mean),
            # whatever the difference leaves (f_2 = 1 and mean is 1 + 1e-6 here); the odd terms of the central
            # difference add h^2 / 6 of it
            d = float(change(t, j, 1e-4) - change(t, j, -1e-4)) / 2e-4
            a = x[t].double().sigmoid()
            u = float((-x[t, j].double()).sigmoid() / a.sum() / T)
            assert abs(d - float(dx[t, j])) <= 2.0 ** -16 * u * float(f[j] + (f * a).sum() / a.sum())


def test_gradient_of_tiny_scores_under_a_large_factor(gpu_available):
    """Scores near 2^-126, whose sum's reciprocal is near 2^126, and a loss that is scaled by 10^6."""
    x = -86.5 + torch.rand(8, 4, generator=torch.Generator().manual_seed(1))
    ids = torch.arange(8, dtype=torch.int32).remainder(3)[:, None]
    grad = torch.tensor([1e6])
    xd = x.to(DEV).requires_grad_(True)
    loss, _ = pkg().balance_loss(xd, ids.to(DEV), None, 1.0)
    dx, = torch.autograd.grad(loss, xd, grad.to(DEV))
    ref, size = _formula(x, ids, torch.tensor([0, 8]), grad, "sigmoid", 1.0)
    assert ((dx.cpu().double() - ref).abs() <= 144 * 2.0 ** -24 * size).all()  # as in test_gradient_of_large_logits


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E", [8, 256])
def test_small_scores_keep_their_precision(gpu_available, score, E):
    """Sequences of one token whose slots all name an expert with a score of
    e^-20 to e^-80: the loss is that score's share, one value each. Logits are
    multiples of 1/8, so that their differences are exact."""
    T = 200
    g = torch.Generator().manual_seed(E)
    x = torch.randint(-8, 9, (T, E), generator=g).float() / 8
    x[:, 3] = -torch.randint(160, 640, (T,), generator=g).float() / 8
    ids = torch.full((T, 1), 3, dtype=torch.int32)
    loss, _ = pkg().balance_loss(x.to(DEV), ids.to(DEV), torch.arange(T + 1, dtype=torch.int32, device=DEV), 1.0, score)
    a = x.double().sigmoid() if score == "sigmoid" else torch.softmax(x.double(), 1)
    want = E * (a / a.sum(1, keepdim=True))[:, 3]
    # half-steps of 2^-24: an exponential 4, sum 1, quotient 4, product 1, of numerator and sum; the sum's E / 32
    # + 5 additions; its reciprocal and the product 2; the store 1
    assert ((loss.cpu().double() - want).abs() <= (28 + E / 32) * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(gpu_available, requires_grad):
    """A dual tensor's tangent is not dropped: the call says that it has no forward-mode derivative."""
    x, ids, off, _ = _inputs(8, 16, 2, 1, torch.float32, 9)
    xd = x.to(DEV).requires_grad_(requires_grad)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        dual = fw.make_dual(xd, torch.ones_like(xd))
        with pytest.raises(RuntimeError, match="forward-mode"):
            pkg().balance_loss(dual, ids.to(DEV), off.to(DEV))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            pkg().balance_loss(dual, ids.to(DEV), off.to(DEV))
        loss, _ = pkg().balance_loss(xd, ids.to(DEV), off.to(DEV))  # no tangent: as ever
    assert torch.equal(loss, pkg().balance_loss(xd, ids.to(DEV), off.to(DEV))[0])
