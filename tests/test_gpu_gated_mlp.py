"""The gated feed-forward block on the tcgen05 kernels against the formula in fp64.

Tolerances count roundings, u = 2^-8 each (half a step of bf16): h, the results and the gradients of the gate and up
columns are rounded once, and the two factors kept for them are off by 2^-10 of themselves.  An error e of an operand
reaches a product as e |other operand|.  fp32 sums are covered by one tenth on top and 1e-5 of the largest value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def _gate(g, act):
    w, dw = g, torch.ones_like(g)
    if act == "gelu":
        c = 2 * math.sqrt(2 / math.pi)
        w, dw = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
    s = torch.sigmoid(w)
    return g * s, s + g * s * (1 - s) * dw


def _oracle(x, wgu, wd, dy, res, act):
    x, wgu, wd, dy = (t.detach().double() for t in (x, wgu, wd, dy))
    g, u = (x @ wgu.t()).chunk(2, 1)
    a, slope = _gate(g, act)
    h = a * u
    y = h @ wd.t() + (0 if res is None else res.detach().double())
    t_y = U * (y.abs() + h.abs() @ wd.abs().t())
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    t_dg, t_du = (U + 2.0 ** -10) * dg.abs(), (U + 2.0 ** -10) * du.abs()
    d, t = torch.cat([dg, du], 1), torch.cat([t_dg, t_du], 1)
    want = [y, d @ wgu, d.t() @ x, dy.t() @ h]
    tol = [t_y, t @ wgu.abs(), t.t() @ x.abs(), U * dy.abs().t() @ h.abs()]
    tol[1:] = [a + U * b.abs() for a, b in zip(tol[1:], want[1:])]
    return want, [1.1 * t + 1e-5 * max(1.0, w.abs().max().item()) for t, w in zip(tol, want)]


def _inputs(m, k, f, n, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + k + f)
    mk = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(torch.bfloat16)  # noqa: E731
    x, wgu, wd = mk(m, k), mk(2 * f, k, std=1.5 / math.sqrt(k)), mk(n, f, std=1 / math.sqrt(f))
    return x, wgu, wd, mk(m, n), (mk(m, n) if residual else None)


def _check(m, k, f, n, act, residual):
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, res = _inputs(m, k, f, n, residual)
    leaves = [t.clone().requires_grad_(True) for t in (x, wgu, wd) + ((res,) if residual else ())]
    y = gemm.gated_mlp(*leaves[:3], act=act, residual=leaves[3] if residual else None)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    want, tol = _oracle(x, wgu, wd, dy, res, act)
    for name, g, w, t in zip(("y", "da", "dw_gate_up", "dw_down"), got, want, tol):
        worst = ((g.double() - w).abs() / t).max().item()
        assert g.shape == w.shape and worst <= 1.0, (name, worst)
    if residual:
        assert torch.equal(got[4], dy)
    with torch.no_grad():
        assert torch.equal(gemm.gated_mlp(x, wgu, wd, act=act, residual=res), y)
    return got


SHAPES = [(1, 8, 8, 8), (7, 64, 64, 72), (8, 1024, 2752, 1024), (33, 136, 200, 136), (128, 256, 128, 64), (129, 72, 1000, 264),
          (300, 768, 136, 768), (16, 512, 72, 8), (64, 40, 2048, 328), (1000, 512, 1376, 512)]


@pytest.mark.parametrize("m,k,f,n", SHAPES)
@pytest.mark.parametrize("act,residual", [("silu", True), ("gelu", False)])
def test_values_and_gradients(m, k, f, n, act, residual):
    _check(m, k, f, n, act, residual)


def test_two_sm_tiles():
    """Long reductions and many tiles take the two-SM kernels in both directions."""
    _check(2500, 1032, 2056, 1096, "silu", True)


def test_extreme_gates():
    """Gates far into both tails: the sigmoid's exponential overflows or vanishes and nothing becomes NaN."""
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, _ = _inputs(40, 64, 64, 64, False)
    for act in ("silu", "gelu"):
        leaves = [(x * 200).requires_grad_(True), wgu.clone().requires_grad_(True), wd.clone().requires_grad_(True)]
        y = gemm.gated_mlp(*leaves, act=act)
        got = [y, *torch.autograd.grad(y, leaves, dy)]
        want, _ = _oracle(leaves[0], wgu, wd, dy, None, act)
        for g, w in zip(got, want):
            assert torch.isfinite(g).all()
            assert ((g.double() - w).norm() / w.norm()).item() < 4 * U


def test_leading_dimensions_strides_and_partial_gradients():
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, res = _inputs(60, 64, 136, 72, True)
    want = gemm.gated_mlp(x, wgu, wd, residual=res)
    got = gemm.gated_mlp(x.view(3, 20, 64), wgu, wd, residual=res.view(3, 20, 72))
    assert got.shape == (3, 20, 72) and torch.equal(got.view(60, 72), want)
    off = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
    for a, w in ((x.t().contiguous().t(), wgu), (off, wgu), (x, wgu.t().contiguous().t())):
        assert torch.equal(gemm.gated_mlp(a, w, wd, residual=res), want)
    leaves = [t.clone().requires_grad_(True) for t in (x, wgu, wd)]
    y = gemm.gated_mlp(*leaves)
    full = torch.autograd.grad(y, leaves, dy)
    for i in range(3):
        some = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        (g,) = torch.autograd.grad(gemm.gated_mlp(*some), [some[i]], dy)
        assert torch.equal(g, full[i])
    y = gemm.gated_mlp(*leaves)
    y.sum().backward()                                                # a gradient without strides of its own
    ones = torch.autograd.grad(gemm.gated_mlp(*leaves), leaves, torch.ones_like(y))
    assert all(torch.equal(t.grad, o) for t, o in zip(leaves, ones))


def test_in_a_captured_graph():
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, res = _inputs(200, 256, 320, 256, True)
    leaves = [t.clone().requires_grad_(True) for t in (x, wgu, wd, res)]
    # no eager graph of the same leaves may live during a capture: autograd would join its stream with the captured one
    want = gemm.gated_mlp(*leaves[:3], residual=leaves[3])
    grads = torch.autograd.grad(want, leaves, dy)
    want = [want.detach(), *grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm.gated_mlp(*leaves[:3], residual=leaves[3])
        grads = torch.autograd.grad(y, leaves, dy)
    for scale in (3, 1):
        with torch.no_grad():
            leaves[0].copy_(x * scale)
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip([y, *grads], want))


def test_gradient_against_differences():
    x, wgu, wd, dy, _ = _inputs(50, 64, 72, 40, False)
    from bluefog_b200.ops import gemm
    for act in ("silu", "gelu"):
        leaves = [t.clone().requires_grad_(True) for t in (x, wgu, wd)]
        grads = torch.autograd.grad(gemm.gated_mlp(*leaves, act=act), leaves, dy)
        torch.manual_seed(2)
        steps = [torch.randn(t.shape, device="cuda", dtype=torch.float64) for t in leaves]

        def loss(e):
            a, b, c = (t.detach().double() + e * s for t, s in zip(leaves, steps))
            g, u = (a @ b.t()).chunk(2, 1)
            return (((_gate(g, act)[0] * u) @ c.t()) * dy.double()).sum().item()

        want = (loss(1e-6) - loss(-1e-6)) / 2e-6
        got = sum((g.double() * s).sum().item() for g, s in zip(grads, steps))
        _, tol = _oracle(x, wgu, wd, dy, None, act)
        bound = math.sqrt(sum((t * s).square().sum().item() for t, s in zip(tol[1:], steps)))       # independent roundings
        assert abs(got - want) <= 4 * bound + 1e-6 * abs(want)


@pytest.mark.parametrize("m", [40, 200])
def test_what_the_kept_factors_cannot_hold(m):
    """Rows with NaN, infinite or huge pre-activations have gradients that are no numbers; the other rows keep theirs."""
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, _ = _inputs(m, 64, 72, 64, False)

    def da(a):
        a = a.clone().requires_grad_(True)
        return torch.autograd.grad(gemm.gated_mlp(a, wgu, wd), a, dy)[0]

    want = da(x)
    bad = x.clone()
    bad[3, 5], bad[17, 0], bad[38] = math.nan, math.inf, x[38] * 1e12
    got = da(bad)
    rows = torch.ones(m, dtype=torch.bool, device="cuda")
    rows[[3, 17, 38]] = False
    assert torch.equal(got[rows], want[rows]) and torch.isfinite(want).all()
    assert got[~rows].isnan().all()


@pytest.mark.parametrize("scale", [2.0 ** -26, 2.0 ** 18])
def test_small_and_large_activations(scale):
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, _ = _inputs(150, 64, 136, 64, False)
    leaves = [(x * scale).requires_grad_(True), wgu.clone().requires_grad_(True), wd.clone().requires_grad_(True)]
    got = torch.autograd.grad(gemm.gated_mlp(*leaves), leaves, dy)
    want, _ = _oracle(leaves[0], wgu, wd, dy, None, "silu")
    for g, w in zip(got, want[1:]):
        assert ((g.double() - w).norm() / w.norm()).item() < 4 * U


def test_gradients_of_gradients_are_refused():
    from bluefog_b200.ops import gemm
    x, wgu, wd, dy, _ = _inputs(40, 64, 72, 64, False)
    x.requires_grad_(True)
    wd.requires_grad_(True)                                           # wgu stays frozen: its gradient is not there
    g, h = torch.autograd.grad(gemm.gated_mlp(x, wgu, wd), [x, wd], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        (g.float().sum() + h.float().sum()).backward()


def test_few_rows_right_behind_the_kernels_that_write_their_inputs():
    """The second product starts beside the first: operands written just before, copies of strided ones and captured launches."""
    from bluefog_b200.ops import gemm
    sets = [_inputs(8, 1024, 1376, 1024, True, seed=s) for s in range(3)]
    want = []
    with torch.no_grad():
        for x, wgu, wd, _, res in sets:
            want.append(gemm.gated_mlp(x, wgu, wd, residual=res))
            torch.cuda.synchronize()
        x, wgu, wd, _, res = (t.clone() for t in sets[0])
        across = wd.t().contiguous().t()
        big = torch.randn(4096, 4096, device="cuda")

        def call():
            return gemm.gated_mlp(x, wgu, wd, residual=res), gemm.gated_mlp(x, wgu, across, residual=res)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = [call() for _ in range(4)]
        for i in (1, 2, 0, 2, 1):
            big = (big @ big).clamp(-1, 1)                            # the host runs ahead of the device
            for t, s in zip((x, wgu, wd, res), (sets[i][0], sets[i][1], sets[i][2], sets[i][4])):
                t.copy_(s)
            across.copy_(sets[i][2])
            eager = [call() for _ in range(4)]
            graph.replay()
            for a, b in zip(eager, y):
                assert all(torch.equal(t, want[i]) for t in (*a, *b))
