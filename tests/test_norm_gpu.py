"""Layer norm, forward and backward, against float64 from the definition."""
import pytest
import torch

from oracle import operators_oracle as O

pytestmark = pytest.mark.gpu


def _bounds(x, w, b, d, eps, G):
    """Element by element, for float32 arithmetic (u = 2^-24, any order of summation, n columns, R rows): the mean is off by n u mean|x|, so x - mean by that and
    a rounding; the variance, a mean of squares about it, by (n + 4) u relative, rstd by half of it and two roundings more.  Sums over n of u = dy w and u xh likewise."""
    u = 2.0 ** -24
    runs = lambda t: t.unflatten(-1, (G, -1))  # noqa: E731
    n = x.shape[-1] // G
    xr = runs(x)
    mean = xr.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((xr - mean) ** 2).mean(-1, keepdim=True) + eps)
    hat = (xr - mean) * r
    e_mean = (n + 2) * u * xr.abs().mean(-1, keepdim=True) + 2 * u * mean.abs()
    e_hat = r * e_mean + hat.abs() * (n + 8) * u                                   # absolute
    w = torch.ones(x.shape[-1], dtype=x.dtype, device=x.device) if w is None else w
    y = e_hat.flatten(-2) * w.abs() + 4 * u * ((hat.flatten(-2) * w).abs() + (0 if b is None else b.abs()))
    if d is None:
        return y, None, None, None
    t = runs(d * w)
    m1, m2 = t.abs().mean(-1, keepdim=True), (t * hat).abs().mean(-1, keepdim=True)
    e1 = (n + 4) * u * m1
    e2 = (n + 4) * u * m2 + (t.abs() * e_hat).mean(-1, keepdim=True)
    inner = t.abs() + m1 + hat.abs() * m2
    dx = r * (e1 + hat.abs() * e2 + e_hat * m2 + (n + 16) * u * inner)
    rows = x.numel() // x.shape[-1]
    d2, h2, e2 = (z.reshape(rows, -1).abs() for z in (d, hat.flatten(-2), e_hat.flatten(-2)))
    return y, dx.flatten(-2), (d2 * e2).sum(0) + (rows + 4) * u * (d2 * h2).sum(0), (rows + 4) * u * d2.sum(0)


def _check(x, w, b, d, eps=1e-5, G=1):
    from flashnystrom_b200 import layer_norm
    lx = x.detach().requires_grad_(True)
    lw, lb = (None if t is None else t.detach().requires_grad_(True) for t in (w, b))
    y = layer_norm(lx, lw, lb, eps, G)
    leaves = [t for t in (lx, lw, lb) if t is not None]
    grads = torch.autograd.grad(y, leaves, d)
    again = torch.autograd.grad(layer_norm(lx, lw, lb, eps, G), leaves, d)
    assert all(torch.equal(p, q) for p, q in zip(grads, again)), "sums are in a fixed order"
    assert torch.equal(layer_norm(x, w, b, eps, G), y), "without a gradient wanted"
    x6 = x.detach().double().requires_grad_(True)
    w6, b6 = (None if t is None else t.detach().double().requires_grad_(True) for t in (w, b))
    ref = O.layer_norm(x6, w6, b6, eps, G)
    refs = torch.autograd.grad(ref, [t for t in (x6, w6, b6) if t is not None], d.double())
    dd = lambda t: None if t is None else t.detach()  # noqa: E731
    bounds = _bounds(x6.detach(), dd(w6), dd(b6), d.double(), eps, G)
    O.within(y, ref, bounds[0], x.dtype)
    O.within(grads[0], refs[0], bounds[1], x.dtype)
    at = 1
    for t, bound in ((w, bounds[2]), (b, bounds[3])):
        if t is not None:
            assert grads[at].dtype == t.dtype
            O.within(grads[at], refs[at], bound, t.dtype)
            at += 1
    return y, grads


def _inputs(rows, cols, dtype, params, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 2 + torch.randn(rows, 1, generator=g)).to(dtype).cuda()
    w, b = ((torch.randn(cols, generator=g) + o).to(params).cuda() for o in (1, 0))
    return x, w, b, torch.randn(rows, cols, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype,params", [(torch.float16, torch.float16), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,cols,G", [
    (1, 1, 1), (3, 2, 1), (1, 512, 1), (7, 8, 1), (5, 17, 1), (1000, 64, 1), (33, 100, 1), (4097, 256, 1), (300, 1000, 1), (130, 1001, 1), (65, 1024, 1), (41, 1025, 1),
    (17, 2048, 1), (9, 4104, 1), (5, 8191, 1), (3, 16384, 1), (2, 16383, 1), (257, 1024, 16), (100, 48, 3), (64, 80, 5), (31, 4096, 64), (9, 8192, 512), (50, 120, 120),
    (20, 4096, 2), (6, 6150, 3), (13, 33 * 7, 7), (3, 36000, 20)])
def test_forward_and_backward(cuda_device, dtype, params, rows, cols, G):
    _check(*_inputs(rows, cols, dtype, params, rows + cols), G=G)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [512, 520, 1024, 1032, 2048, 2056, 4096, 4100, 8192, 8200, 16376])
def test_lengths_around_what_threads_hold(cuda_device, dtype, cols):
    _check(*_inputs(1200, cols, dtype, torch.float32, cols))


@pytest.mark.parametrize("cols,G", [(512, 1), (512, 8), (3000, 1)])
def test_without_weight_or_bias(cuda_device, cols, G):
    x, w, b, d = _inputs(37, cols, torch.float16, torch.float32, 3)
    _check(x, None, None, d, G=G)
    _check(x, w, None, d, G=G)
    _check(x, None, b, d, G=G)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G", [1, 4])
def test_shapes_and_strides(cuda_device, dtype, G):
    """Leading dimensions, rows apart, a start and a row distance off sixteen bytes, orders that are copied, a gradient that is spread out of one value."""
    x, w, b, d = _inputs(60, 256, dtype, torch.float32, 5)
    y, grads = _check(x, w, b, d, G=G)
    y3, g3 = _check(x.view(3, 4, 5, 256), w, b, d.view(3, 4, 5, 256), G=G)
    assert torch.equal(y3.view(60, 256), y) and torch.equal(g3[1], grads[1])
    apart = torch.zeros(60, 300, dtype=dtype, device="cuda")
    for off in (0, 8, 1):
        view = apart[:, off:off + 256]
        view.copy_(x)
        _check(view, w, b, d, G=G)
    odd = torch.zeros(60, 257, dtype=dtype, device="cuda")[:, 1:]
    odd.copy_(d)
    _check(x, w, b, odd, G=G)
    turned = x.view(5, 12, 256).transpose(0, 1)
    _check(turned, w, b, d.view(12, 5, 256), G=G)
    _check(x, w, b, torch.ones(1, 1, dtype=dtype, device="cuda").expand(60, 256), G=G)
    _check(x[:1].expand(60, 256), w, b, d, G=G)
    wide = torch.zeros(513, device="cuda")
    wide[1::2] = w
    _check(x, wide[1::2], b, d, G=G)
    _check(x[0], w, b, d[0], G=G)


def test_values(cuda_device):
    """Rows of one value, rows far from zero, tiny and huge spreads, eps of zero; infinities stay in their row."""
    from flashnystrom_b200 import layer_norm
    x, w, b, d = _inputs(40, 512, torch.float32, torch.float32, 9)
    x[0], x[1], x[2], x[3] = 3.0, x[1] + 1000.0, x[2] * 1e-4, x[3] * 1e8
    _check(x, w, b, d)
    _check(x[1:], w, b, d[1:], eps=0.0)
    _check(x, w, b, d, eps=0.1)
    clean = layer_norm(x, w, b)
    x[7, 3], x[9, 0] = float("inf"), float("nan")
    y = layer_norm(x, w, b)
    others = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[others], clean[others]) and not torch.isfinite(y[7]).any() and torch.isnan(y[9]).all()


def test_many_rows(cuda_device):
    """More rows than places: every CTA goes round; sums over 70000 rows."""
    _check(*_inputs(70001, 64, torch.bfloat16, torch.float32, 1))
    _check(*_inputs(20000, 1024, torch.float16, torch.float16, 2), G=16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols,G", [(3, 1), (17, 1), (27, 3), (101, 1), (250, 1), (501, 3), (513, 1), (66, 22), (700, 28)])
def test_many_rows_of_odd_lengths(cuda_device, dtype, cols, G):
    """Rows that loads of 16 bytes do not divide, far more of them than the device has places: each place's rows begin as far into 16 bytes."""
    rows = 40000 if cols < 200 else 9001
    x, w, b, d = _inputs(rows, cols, dtype, torch.float32, cols)
    _check(x, w, b, d, G=G)
    apart = torch.zeros(2, rows * (cols + 5) + 9, dtype=dtype, device="cuda")
    views = [t[3:3 + rows * (cols + 5)].view(rows, cols + 5)[:, 2:2 + cols] for t in apart]
    views[0].copy_(x)
    views[1].copy_(d)
    _check(views[0], w, b, views[1], G=G)


def test_gradients_against_differences(cuda_device):
    """Central differences of the float32 call: truncation h^2 / 6 times a third derivative of order one, rounding 2^-22 / h."""
    from flashnystrom_b200 import layer_norm
    x, w, b, d = _inputs(16, 128, torch.float32, torch.float32, 4)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves, num_groups=2), leaves, d)
    h = 1e-2
    for i, g in enumerate(grads):
        e = torch.randn_like(leaves[i])
        f = lambda s: (layer_norm(*(t.detach() + (s * h * e if j == i else 0) for j, t in enumerate(leaves)), num_groups=2).double() * d).sum()  # noqa: E731
        diff = float((f(1) - f(-1)) / (2 * h))
        assert abs(float((g.double() * e).sum()) - diff) <= 2e-4 * float((g.double() * e).norm()) * 16 ** 0.5 + 2e-2


def test_streams_graphs_and_wanted_parts(cuda_device):
    from flashnystrom_b200 import layer_norm
    x, w, b, d = _inputs(3000, 768, torch.float16, torch.float32, 6)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves, num_groups=12)
        return [y.detach(), *torch.autograd.grad(y, leaves, d)]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        leaves[0].mul_(-1.5)
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, step()))
    full = step()
    for i, t in enumerate(leaves):
        args = [s.detach() if j != i else s for j, s in enumerate(leaves)]
        (g,) = torch.autograd.grad(layer_norm(*args, num_groups=12), t, d)
        assert torch.equal(g, full[1 + i])
    (g,) = torch.autograd.grad(layer_norm(*leaves), leaves[0], d, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), leaves[0])


def test_module_and_empty(cuda_device):
    from flashnystrom_b200 import LayerNorm, layer_norm
    m, t = LayerNorm(512).cuda(), torch.nn.LayerNorm(512).cuda()
    with torch.no_grad():
        t.weight.normal_()
        t.bias.normal_()
    m.load_state_dict(t.state_dict())
    x = torch.randn(3, 5, 512, device="cuda")
    assert torch.allclose(m(x), t(x), rtol=1e-5, atol=1e-5)
    m(x).sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None
    w = torch.ones(512, device="cuda", requires_grad=True)
    y = layer_norm(x[:0], w)
    y.sum().backward()
    assert y.shape == (0, 5, 512) and not w.grad.any()


def test_refusals(cuda_device):
    from flashnystrom_b200 import LayerNorm, layer_norm
    x = torch.randn(4, 64, device="cuda", dtype=torch.float16)
    w = torch.ones(64, device="cuda")
    for message, call in [("no CPU path", lambda: layer_norm(x.cpu())), ("must divide", lambda: layer_norm(x, num_groups=3)), ("must divide", lambda: layer_norm(x, num_groups=0)),
                          ("64 values", lambda: layer_norm(x, w[:32])), ("must be float32 or", lambda: layer_norm(x, w.bfloat16())),
                          ("dtypes must match", lambda: layer_norm(x, w, w.half())), ("Supported dtypes", lambda: layer_norm(x.double())), ("eps must be", lambda: layer_norm(x, eps=-1.0)),
                          ("must be a CUDA tensor", lambda: layer_norm(x, w.cpu())), ("at most 16384", lambda: layer_norm(torch.zeros(2, 16400, device="cuda"))),
                          ("last dimension must be", lambda: LayerNorm(32).cuda()(x)), ("last dimension to normalise", lambda: layer_norm(x[:, :0]))]:
        with pytest.raises(RuntimeError, match=message):
            call()
