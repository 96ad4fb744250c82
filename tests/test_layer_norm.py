"""Layer norm (ops/functional.py) against a plain 64-bit form.

Tolerances, fixed beforehand.  fp32 sums of C terms in any order are off by at
most C 2^-24 of the sum of magnitudes.  With A = max |x| of a row and std its
sqrt(var + eps): the mean is off by C 2^-24 A, a distance by that and 2^-24 A,
so h = (x - mean) / std by (C + 4) 2^-24 A / std and, through the variance (a
sum of C squares, then a root and a product), by (C + 8) 2^-24 |h| more.  The
worst case of every sum at once is far from what happens, and these bounds are
still some 1e-3 at most here.  The backward pass adds two means of C terms of
|g| and |g h|; every result ends with its own rounding, eps / 2."""

import pytest
import torch

from rainbowiqn_amd.ops import functional as F

gpu = pytest.mark.gpu
U = 2.0 ** -24


def plain(x, w, b, eps, dy=None):
    """y, dx, dw, db and bounds for them, in 64 bits on the CPU."""
    x = x.detach().double().cpu()
    c = x.shape[1]
    w = torch.ones(c).double() if w is None else w.detach().double().cpu()
    b = torch.zeros(c).double() if b is None else b.detach().double().cpu()
    d = x - x.mean(1, keepdim=True)
    std = ((d * d).mean(1, keepdim=True) + eps).sqrt()
    h = d / std
    eh = (c + 4) * U * x.abs().amax(1, keepdim=True) / std + (c + 8) * U * h.abs()
    out = {"y": (h * w + b, eh * w.abs() + 4 * U * ((h * w).abs() + b.abs()))}
    if dy is not None:
        dy = dy.detach().double().cpu()
        g = dy * w
        c2 = (g * h).mean(1, keepdim=True)
        dx = (g - g.mean(1, keepdim=True) - h * c2) / std
        mag = g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (
            g * h).abs().mean(1, keepdim=True)
        e = (c + 12) * U * mag + eh * c2.abs() + h.abs() * (
            g.abs() * eh).mean(1, keepdim=True)
        rel_std = (c + 8) * U + ((c + 4) * U * x.abs().amax(1, keepdim=True) / std) ** 2
        out["dx"] = (dx, e / std + rel_std * dx.abs())
        r = x.shape[0]
        out["dw"] = ((dy * h).sum(0), (r + 4) * U * (dy * h).abs().sum(0)
                     + (dy.abs() * eh).sum(0))
        out["db"] = (dy.sum(0), (r + 4) * U * dy.abs().sum(0))
    return out


def near(got, want, bound):
    assert got.shape == want.shape
    tiny = torch.finfo(got.dtype).smallest_normal
    off = ((got.detach().double().cpu() - want).abs() - bound
           - torch.finfo(got.dtype).eps / 2 * (want.abs() + bound) - tiny)
    assert bool((off <= 0).all()), float(off.max())


def inputs(r, c, dtype, wdtype, device, offset=0.3):
    g = torch.Generator().manual_seed(r * 10007 + c)
    x = (torch.randn(r, c, generator=g) + offset) * torch.exp(
        torch.randn(r, 1, generator=g))
    w = 1 + 0.5 * torch.randn(c, generator=g)
    b = torch.randn(c, generator=g)
    dy = torch.randn(r, c, generator=g)
    return (x.to(dtype).to(device).requires_grad_(),
            w.to(wdtype).to(device).requires_grad_(),
            b.to(wdtype).to(device).requires_grad_(), dy.to(dtype).to(device))


def step(x, w, b, dy, eps=1e-5):
    y = F.layer_norm(x, w, b, eps)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db"), (x, w, b))
                      if t is not None], torch.autograd.grad(y, leaves, dy)))
    return {"y": y, **grads}


SHAPES = [(1, 1), (1, 3136), (3, 2), (5, 8), (7, 511), (64, 512), (33, 513),
          (130, 1024), (129, 1537), (2050, 200), (257, 3136), (50, 4096),
          (9, 4097), (300, 5000), (2, 40000)]
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32)]


@pytest.mark.parametrize("shape", [(1, 1), (7, 33), (20, 300)])
def test_cpu(shape):
    x, w, b, dy = inputs(*shape, torch.float32, torch.float32, "cpu")
    got = step(x, w, b, dy)
    for name, (want, bound) in plain(x, w, b, 1e-5, dy).items():
        near(got[name], want, bound)


def test_formula_against_differences():
    """The plain form's gradients against central differences in 64 bits: off by
    h^2 (1e-10) of third derivatives of order 10 and 1e-16 / h of the loss."""
    x, w, b, dy = inputs(3, 17, torch.float32, torch.float32, "cpu")
    out = plain(x, w, b, 1e-5, dy)
    args = [t.detach().double() for t in (x, w, b)]
    loss = lambda: float((plain(*args, 1e-5)["y"][0] * dy.double()).sum())  # noqa: E731
    for t, name, places in ((args[0], "dx", [(0, 0), (1, 9), (2, 16)]),
                            (args[1], "dw", [(0,), (16,)]),
                            (args[2], "db", [(0,), (16,)])):
        for at in places:
            keep = float(t[at])
            t[at] = keep + 1e-5
            up = loss()
            t[at] = keep - 1e-5
            down = loss()
            t[at] = keep
            assert abs((up - down) / 2e-5 - float(out[name][0][at])) < 1e-7


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_step(shape, types):
    x, w, b, dy = inputs(*shape, *types, "cuda")
    got = step(x, w, b, dy)
    for name, (want, bound) in plain(x, w, b, 1e-5, dy).items():
        near(got[name], want, bound)
    assert got["dw"].dtype == types[1] and got["dx"].dtype == types[0]
    with torch.no_grad():
        assert torch.equal(F.layer_norm(x, w, b), got["y"])


@gpu
@pytest.mark.parametrize("which", [(0, 0), (1, 0), (0, 1)])
@pytest.mark.parametrize("cols", [300, 4500])
def test_without_weight_or_bias(cols, which):
    x, w, b, dy = inputs(40, cols, torch.float32, torch.float32, "cuda")
    w, b = w if which[0] else None, b if which[1] else None
    got = step(x, w, b, dy)
    want = plain(x, w, b, 1e-5, dy)
    for name in got:
        near(got[name], *want[name])


@gpu
@pytest.mark.parametrize("cols", [64, 3136, 4100])
def test_rows_that_are_hard(cols):
    """A large offset keeps its digits, equal values give the bias, and what is
    not finite stays in its row."""
    x, w, b, dy = inputs(8, cols, torch.float32, torch.float32, "cuda")
    with torch.no_grad():
        x[1] += 1000.0
        x[2] = 5.0
        x[3, 7] = float("inf")
        x[4, 9] = float("nan")
        x[5] = 0.0
        x[6] *= 1e15
    got = step(x, w, b, dy)
    fine = [0, 1, 2, 5, 6, 7]
    want = plain(x[fine], w, b, 1e-5, dy[fine])
    for name in ("y", "dx"):
        near(got[name][fine], *want[name])
        assert got[name][3:5].isnan().all()
    assert torch.equal(got["y"][2], b.detach())
    assert got["db"].isfinite().all()


@gpu
@pytest.mark.parametrize("cols", [504, 4600])
def test_views(cols):
    base = torch.randn(60, 2 * cols + 16, device="cuda").to(torch.bfloat16)
    w = torch.randn(cols, device="cuda").to(torch.bfloat16)
    for x in (base[:, 1:cols + 1], base[::3, 8:cols + 8], base[:, :2 * cols:2],
              base[:1, :cols].expand(17, cols), base[:, :cols].t()[:60].t()):
        want = F.layer_norm(x.contiguous(), w[:x.shape[1]].contiguous())
        assert torch.equal(F.layer_norm(x, w[:x.shape[1]].contiguous()), want)
    x = base[:, 3:cols + 3].detach().requires_grad_()
    y = F.layer_norm(x.view(5, 12, cols) if x.is_contiguous() else x, w)
    y.sum().backward()  # a gradient that is one number spread out
    near(x.grad, *plain(x, w, None, 1e-5, torch.ones_like(y))["dx"])
    # weights that are not 16-byte aligned
    w1 = torch.randn(cols + 1, device="cuda")[1:]
    x = base[:, :cols]
    near(F.layer_norm(x, w1), *plain(x, w1, None, 1e-5)["y"])
    # leading dimensions
    x3 = base[:, :cols].reshape(3, 4, 5, cols)
    assert torch.equal(F.layer_norm(x3, w).view(60, cols), F.layer_norm(x, w))
    assert torch.equal(F.layer_norm(x[7], w), F.layer_norm(x, w)[7])


def refusals(device):
    x, w = torch.randn(4, 30, device=device), torch.randn(30, device=device)
    for call in (lambda: F.layer_norm(x, w[:29]),
                 lambda: F.layer_norm(x, None, w[:29]),
                 lambda: F.layer_norm(x, w.view(1, 30)),
                 lambda: F.layer_norm(x, w, eps=-1.0),
                 lambda: F.layer_norm(x, w, eps=float("nan")),
                 lambda: F.layer_norm(x, w.bfloat16()),
                 lambda: F.layer_norm(x.bfloat16(), w, w.bfloat16()),
                 lambda: F.layer_norm(x.long(), w),
                 lambda: F.layer_norm(x[:, :0]),
                 lambda: F.layer_norm(x[0, 0])):
        with pytest.raises(RuntimeError):
            call()


def test_refusals_cpu():
    refusals("cpu")


@gpu
def test_refusals_gpu():
    refusals("cuda")
    x, w = torch.randn(4, 30, device="cuda"), torch.randn(60, device="cuda")
    for call in (lambda: F.layer_norm(x, w.cpu()[:30]),
                 lambda: F.layer_norm(x, w[::2])):
        with pytest.raises(RuntimeError):
            call()
    x.requires_grad_()
    y = F.layer_norm(x)
    (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_no_rows(device):
    x = torch.zeros(0, 40, device=device, requires_grad=True)
    w = torch.ones(40, device=device, requires_grad=True)
    y = F.layer_norm(x, w, w)
    y.sum().backward()
    assert y.shape == x.grad.shape == (0, 40) and not w.grad.any()


@gpu
def test_parts_of_the_gradient_and_same_bits():
    x, w, b, dy = inputs(700, 1000, torch.bfloat16, torch.float32, "cuda")
    whole = torch.autograd.grad(F.layer_norm(x, w, b), (x, w, b), dy)
    for want in ([0], [1], [2], [0, 2], [1, 2]):
        args = [t.detach().clone().requires_grad_(i in want)
                for i, t in enumerate((x, w, b))]
        grads = torch.autograd.grad(F.layer_norm(*args), [args[i] for i in want], dy)
        for i, g in zip(want, grads):
            assert torch.equal(g, whole[i])


@gpu
def test_captured_step_replays():
    graphs = []
    for shape in ((256, 3136), (40, 5000)):
        x, w, b, dy = inputs(*shape, torch.bfloat16, torch.bfloat16, "cuda")
        one = lambda x=x, w=w, b=b, dy=dy: [  # noqa: E731
            t.detach() for t in step(x, w, b, dy).values()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = one()
        graphs.append((graph, outs, x, one))
    for i in range(4):
        for graph, outs, x, one in graphs:
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, one()))


@gpu
def test_offsets_past_32_bits():
    rows, cols = 2 ** 20 + 3, 2056
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    tail, w, b, dy = inputs(50, cols, torch.bfloat16, torch.bfloat16, "cuda")
    x[-50:] = tail.detach()
    x.requires_grad_()
    y = F.layer_norm(x, w, b)
    assert torch.equal(y[-50:], F.layer_norm(tail, w, b))
    g = torch.zeros_like(y)
    g[-50:] = dy
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    got = {"dx": dx[-50:], "dw": dw, "db": db}
    want = plain(tail, w, b, 1e-5, dy)
    for name in got:
        near(got[name], *want[name])
    assert not dx[:-50].any()


def changed_in_place(device):
    """A result may be changed in place, like any other."""
    x = torch.randn(6, 40, device=device, requires_grad=True)
    w = torch.randn(40, device=device, requires_grad=True)
    for shape in ((6, 40), (2, 3, 40)):
        want = torch.relu(F.layer_norm(x.view(shape), w) * 2)
        got = F.layer_norm(x.view(shape), w).mul_(2).relu_()
        assert torch.equal(got, want)
        for p, q in zip(torch.autograd.grad(got.sum(), (x, w)),
                        torch.autograd.grad(want.sum(), (x, w))):
            assert torch.equal(p, q)


def test_changed_in_place_cpu():
    changed_in_place("cpu")


@gpu
def test_changed_in_place_gpu():
    changed_in_place("cuda")


@gpu
def test_capture_beside_an_eager_graph_is_refused():
    x = torch.randn(6, 200, device="cuda", requires_grad=True)
    w = torch.randn(200, device="cuda", requires_grad=True)
    call = lambda: F.layer_norm(x, w)  # noqa: E731
    alive = call()  # holds the leaves' nodes, which are of the default stream
    dy = torch.ones_like(alive)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
        with pytest.raises(RuntimeError, match="captured"):
            torch.autograd.grad(y, (x, w), dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive)
    alive.backward(dy)  # that one is as before
    assert x.grad.shape == x.shape


@gpu
def test_most_columns():
    x = torch.randn(2, 2 ** 24, device="cuda").bfloat16().requires_grad_()
    w = torch.rand(2 ** 24, device="cuda").requires_grad_()
    dy = torch.randn(2, 2 ** 24, device="cuda").bfloat16()
    F.layer_norm(x, w).backward(dy)
    h = x.detach().double()
    h = h - h.mean(1, keepdim=True)
    h = h / (h.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
    # sums of 2^24 terms of either sign in fp32, by 256 threads of 2^16 each,
    # leave mean and rstd 2^16 x 2^-24 of a term off at the very most
    want = (dy.double() * h).sum(0)
    off = (w.grad.double() - want).abs()
    assert bool((off <= 2.0 ** -7 * (dy.double() * h).abs().sum(0) + 2.0 ** -7
                 * dy.double().abs().sum(0)).all())
    with pytest.raises(RuntimeError):
        F.layer_norm(torch.empty(1, 2 ** 24 + 1, device="cuda"))


@gpu
@pytest.mark.parametrize("cols", [8, 520, 1001, 1040, 2056, 4104])
def test_infinite_weight_stays_in_its_column(cols):
    """y and dw of the others are finite.  Both means of dx are infinite, mean(g)
    with the sign of dy there and mean(g h) with h's as well, so
    g - mean(g) - h mean(g h) is infinite where h has the sign of that column's
    and NaN where it has the other."""
    x = torch.randn(5, cols, device="cuda", requires_grad=True)
    w = torch.ones(cols, device="cuda")
    w[-1] = float("inf")
    w.requires_grad_()
    dy = torch.randn(5, cols, device="cuda")
    y = F.layer_norm(x, w)
    assert y[:, :-1].isfinite().all() and y[:, -1].isinf().all()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.isfinite().all()
    h = x - x.mean(1, keepdim=True)
    same = (h * h[:, -1:] > 0)[:, :-1]
    assert torch.equal(dx[:, :-1].isnan(), ~same)
    assert dx[:, :-1][same].isinf().all()


@gpu
@pytest.mark.parametrize("types", [(torch.float32,) * 2, (torch.bfloat16,) * 2,
                                   (torch.float16, torch.float32)])
@pytest.mark.parametrize("cols", [1, 7, 8, 9, 15, 503, 505, 511, 513, 1023, 1025,
                                  2047, 2049, 4089, 4095, 4097])
def test_odd_columns(cols, types):
    """Rows whose end and beginning lie anywhere, where two lanes have the last
    columns."""
    wide, w, b, wide_dy = inputs(37, cols + 3, *types, "cuda")
    x = wide.detach()[:, 3:].requires_grad_()
    w, b = (t.detach()[3:].clone().requires_grad_() for t in (w, b))
    dy = wide_dy[:, 1:cols + 1]
    got = step(x, w, b, dy)
    for name, (want, bound) in plain(x, w, b, 1e-5, dy).items():
        near(got[name], want, bound)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [4097, 32768, 100001, 2 ** 20, 2 ** 24])
def test_long_rows_keep_their_digits(cols, dtype):
    """Rows of one large number, of a large offset and around zero, with a
    gradient that is one number and one of either sign.

    Sums go by runs of 256 columns a thread, then of the runs, then over 256
    threads: n = 256 + cols / 2^16 + 10 additions one behind the other, off by
    n 2^-24 of the magnitudes.  The first mean is off by e0 = n U A, A = max |x|.
    The distances' sum mends that up to em = U A (the mean's own rounding) +
    n U (mean |d| + e0), and the variance is off by (n + 4) U of the mean of
    (|d| + e0)^2, twice that for the square that is taken off, and em^2."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = normal(3, cols)
    x[0] = 1000.1
    x[1] += 1000.0
    x = x.to(dtype).requires_grad_()
    w = (1 + 0.1 * normal(cols)).requires_grad_()
    dy = 0.1 * normal(3, cols)
    dy[1] = 0.1
    dy = dy.to(dtype)
    with torch.no_grad():
        w[:] = torch.where(torch.arange(cols, device="cuda") % 2 == 0, w, 1.0)
    got = {"y": F.layer_norm(x, w)}
    got["dx"], got["dw"] = torch.autograd.grad(got["y"], (x, w), dy)
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    n, xd, wd, dyd = 266 + cols / 2 ** 16, x.detach().double(), w.detach().double(), dy.double()
    d = xd - mean(xd)
    var = mean(d * d) + 1e-5
    std = var.sqrt()
    h = d / std
    top = xd.abs().amax(1, keepdim=True)
    e0 = n * U * top
    em = U * top + n * U * (mean(d.abs()) + e0)
    rel = ((n + 4) * U * 3 * mean((d.abs() + e0) ** 2) + em ** 2) / (2 * var) + 4 * U
    eh = (em + U * d.abs()) / std + rel * h.abs()
    gw = dyd * wd
    c1, c2 = mean(gw), mean(gw * h)
    want = {"y": (h * wd, eh * wd.abs() + 2 * U * (h * wd).abs()),
            "dw": ((dyd * h).sum(0), (dyd.abs() * eh).sum(0)
                   + 4 * U * (dyd * h).abs().sum(0))}
    off = (4 * U * (gw.abs() + c1.abs() + (h * c2).abs()) + n * U * mean(gw.abs())
           + h.abs() * (n * U * mean((gw * h).abs()) + mean(gw.abs() * eh))
           + eh * c2.abs())
    dx = (gw - c1 - h * c2) / std
    want["dx"] = (dx, off / std * (1 + rel) + rel * dx.abs())
    for name, (value, bound) in want.items():
        near(got[name], value.cpu(), bound.cpu())


@gpu
@pytest.mark.parametrize("rows,cols", [(2 ** 24 - 3, 8), (2 ** 24 + 5, 3),
                                       (2 ** 21 + 1, 1032), (2 ** 22, 300)])
def test_sums_over_many_rows(rows, cols):
    """A gradient that is one number, and a column whose h has one sign.  A
    register adds up 256 rows and 4 more of its last round; or 256 and then rows /
    2^17 runs, of which 512 workgroups are left for 256 rows each; 64 parts, then
    their runs and 16 shares.  4 waves and a rounding: 8 more."""
    torch.manual_seed(rows)
    x = torch.randn(rows, cols, device="cuda")
    x[:, 0] += 50.0
    w = torch.ones(cols, device="cuda", requires_grad=True)
    b = torch.zeros(cols, device="cuda", requires_grad=True)
    dy = torch.full((1, cols), 0.1, device="cuda").expand(rows, cols)
    dw, db = torch.autograd.grad(F.layer_norm(x, w, b), (w, b), dy)
    n = 260 + rows / 2 ** 17 + 64 + 16 + 8
    if cols >= 8:  # parts: of 256 rows for each of a workgroup's teams
        n = 260 + 64 + rows / 256 / (4 if cols <= 1024 else 1) / 2 ** 10 + 16 + 8
    one = float(dy[0, 0].double())
    assert bool(((db.double() - one * rows).abs() <= n * U * one * rows).all())
    var, mean = torch.var_mean(x.double(), 1, unbiased=False)
    std = (var + 1e-5).sqrt()
    for c in (0, 1, cols - 1):
        h = (x[:, c].double() - mean) / std
        top = x.abs().amax(1).double()
        eh = (cols + 4) * U * top / std + (cols + 8) * U * h.abs()
        bound = (n * U * h.abs() + eh).sum() * one
        if c == 0:  # h is off by some 2^-24 either way, row by row: of 2^21 rows
            # and more 1 % of the worst case is far from what is left
            bound = (n * U * h.abs() + 0.01 * eh).sum() * one
        assert float((dw[c].double() - one * h.sum()).abs()) <= float(bound)


def duals(x, w, b):
    from torch.autograd import forward_ad

    for i in range(3):
        args = [x, w, b]
        args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
        yield i, F.layer_norm, args


@gpu
@pytest.mark.parametrize("cols", [30, 5000])
def test_tangents_are_refused(cols):
    """Instead of a result without one, which would count as zero."""
    from torch.autograd import forward_ad

    x, w, b, _ = inputs(4, cols, torch.float32, torch.float32, "cuda")
    for leaves in ((x, w, b), tuple(t.detach() for t in (x, w, b))):
        with forward_ad.dual_level():
            for _, call, args in duals(*leaves):
                for mode in (torch.no_grad, torch.enable_grad):
                    with mode(), pytest.raises(RuntimeError):
                        call(*args)
            F.layer_norm(*leaves)


def test_tangents_cpu():
    """There the derivative in x's, weight's and bias's direction is right."""
    from torch.autograd import forward_ad

    x, w, b, _ = (t.detach() for t in inputs(4, 30, torch.float32, torch.float32, "cpu"))
    d = x.double() - x.double().mean(1, keepdim=True)
    h = d / ((d * d).mean(1, keepdim=True) + 1e-5).sqrt()
    # x moved by one number: y stays; weight by 1: h; bias by 1: 1
    want = [torch.zeros_like(h), h, torch.ones_like(h)]
    with forward_ad.dual_level():
        for i, call, args in duals(x, w, b):
            got = forward_ad.unpack_dual(call(*args)).tangent
            assert bool(((got.expand_as(h).double() - want[i]).abs() <= 1e-5).all())


@gpu
@pytest.mark.parametrize("cols", [64, 3136, 4100, 40000])
def test_variances_past_the_range(cols):
    """Squares past fp32's range make the variance infinite and h zero, as in the
    plain form in fp32: y is the bias and nothing comes back but the bias's
    gradient."""
    x = 1e32 * (1 + torch.rand(3, cols, device="cuda"))
    x[1, ::2] *= -1
    x.requires_grad_()
    w = torch.randn(cols, device="cuda", requires_grad=True)
    b = torch.randn(cols, device="cuda", requires_grad=True)
    y = F.layer_norm(x, w, b)
    assert torch.equal(y, b.detach().expand_as(y))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert not dx.any() and not dw.any() and torch.equal(db, torch.full_like(db, 3.0))
    # one number in every place: y stays finite, however far the mean is off
    const = torch.full((1, cols), 1e32, device="cuda")
    assert F.layer_norm(const, w, b).isfinite().all()
