"""GPU tests of linear_act (csrc/linear.hip) against the formulas in 64 bits.

Tolerances, u = 2^-24.  h = x w^T + b is a sum of K products: 16-bit products are exact in fp32, each
sum adds at most u of what is summed so far (any order: (K + splits) u sum |x||w|, far from reached; the
bound below uses min(K, 64) + 8 + K / 64 for sums that run 32 k at a time per instruction);
float32 adds 2^-22 sum |x||w| for the parts left out and the six products' own sums.  An activation's
slope is at most 1.13, its own error 4 u |.| + 4 u.  Results are rounded by half a step of the type;
the backward starts from h (dh) rounded once to the type: half a step of it, relative, into
every product with it, and half a step of h times |act''| <= 1 into dh."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLOATS = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "gelu", "silu", "sigmoid", "tanh"]


def _F():
    from lvmhelpers import functional
    return functional


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _sum_err(K, dtype):
    return U * (min(K, 64) + 8 + K / 64 + (4 + 6 * (min(K, 64) + 8 + K / 64) / 16 if dtype == torch.float32 else 0))


def _act(name, h):
    return {"none": lambda: h, "relu": lambda: h.clamp_min(0), "gelu": lambda: torch.nn.functional.gelu(h),
            "silu": lambda: torch.nn.functional.silu(h), "sigmoid": lambda: torch.sigmoid(h),
            "tanh": lambda: torch.tanh(h)}[name]()


def _case(M, N, K, dtype, seed, bias=True, res=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return ((r(M, K)).to(dtype), (r(N, K) * max(K, 1) ** -0.5).to(dtype), (r(N) * 0.5).to(dtype) if bias else None,
            r(M, N).to(dtype) if res else None, r(M, N).to(dtype))


def _within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))


def _check(dev, x, w, b, r, dy, act, dtype, run=None, grads=True):
    M, K = x.shape
    N = w.shape[0]
    leaves = [None if t is None else t.to(dev).requires_grad_(grads) for t in (x, w, b, r)]
    y = (run or _F().linear_act)(leaves[0], leaves[1], leaves[2], act, leaves[3])
    # the reference, on the GPU in fp64 where it is large
    where = dev if M * N * K > 1 << 24 else "cpu"
    X, W, B, R, DY = (None if t is None else t.to(where).double() for t in (x, w, b, r, dy))
    h = X @ W.t().contiguous()
    mag = X.abs() @ W.abs().t().contiguous()
    if B is not None:
        h, mag = h + B, mag + B.abs()
    h = h.requires_grad_(True)
    a = _act(act, h)
    want = a + (R if R is not None else 0)
    half = _half(dtype) if dtype != torch.float32 else U
    herr = _sum_err(K, dtype) * mag
    aerr = 1.13 * herr + 8 * U * (a.detach().abs() + 1 * (act not in ("none", "relu")))
    _within(y.detach(), want.detach().cpu(), (aerr + half * want.detach().abs() * 1.01 + 2 * U * (R.abs() if R is not None else 0) + 2.0 ** -25 * (dtype == torch.float16)).cpu())
    if not grads:
        return
    (dh,) = torch.autograd.grad(a, h, DY)
    hd = h.detach()
    near = (hd.abs() <= herr).double() if act == "relu" else 0.0        # relu's corner may fall either way
    # dh: slope at the rounded h, then rounded
    dherr = DY.abs() * (1.01 * (herr + half * hd.abs() * (dtype != torch.float32)) * (act not in ("none", "relu")) + 12 * U + near) + half * dh.abs() * (
        dtype != torch.float32 and act != "none") + 2.0 ** -25 * (dtype == torch.float16)
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(dev))
    got = iter(got)
    Wc, Xc = W.contiguous(), X
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -120
    want_dx = dh @ Wc
    _within(next(got), want_dx.cpu(), (dherr @ Wc.abs() + _sum_err(N, dtype) * (dh.abs() @ Wc.abs()) + half * want_dx.abs() * 1.01 + tiny).cpu())
    dht = dh.t().contiguous()
    want_dw = dht @ Xc
    _within(next(got), want_dw.cpu(), (dherr.t().contiguous() @ Xc.abs() + _sum_err(M, dtype) * (dht.abs() @ Xc.abs()) + half * want_dw.abs() * 1.01 + tiny).cpu())
    if b is not None:
        want_db = dh.sum(0)
        _within(next(got), want_db.cpu(), (dherr.sum(0) + _sum_err(M, dtype) * dh.abs().sum(0) + half * want_db.abs() * 1.01 + tiny).cpu())
    if r is not None:
        assert torch.equal(next(got).cpu(), dy)


# below, at and over every tile and fragment edge; odd widths take the unaligned path
SIZES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 64, 64), (17, 16, 32), (64, 64, 64), (65, 63, 66), (128, 128, 128),
         (127, 129, 257), (200, 72, 1000), (1, 4096, 512), (3, 1000, 777), (5000, 8, 16), (4097, 24, 40), (300, 784, 16),
         (33, 1024, 8), (256, 256, 72)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_every_size(dev, M, N, K, dtype):
    _check(dev, *_case(M, N, K, dtype, M + N + K), "gelu", dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,res", [(True, True), (False, False), (False, True)])
def test_every_epilogue(dev, act, bias, res, dtype):
    for M, N, K in ((70, 96, 48), (70, 97, 47)):
        _check(dev, *_case(M, N, K, dtype, 5, bias, res), act, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 128), (4160, 4352, 200), (2048, 2048, 1024), (1, 64, 70000), (20000, 16, 24)])
def test_large_tiles_and_long_sums(dev, M, N, K, dtype):
    """The 256 x 256 and 128 x 128 tiles (full and partly filled), and products split over a long axis."""
    _check(dev, *_case(M, N, K, dtype, 1), "silu", dtype)


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 2048), (4100, 4090, 2050), (9000, 260, 9000)])
def test_the_widest_fp32_tiles(dev, M, N, K):
    """256 x 128 tiles with the next tile split while one is multiplied, full and partly filled."""
    _check(dev, *_case(M, N, K, torch.float32, 1), "none", torch.float32)


def test_fp32_keeps_fp32_accuracy(dev):
    """Values over 60 binades and sums that cancel: three bf16 parts carry all 24 bits."""
    g = torch.Generator().manual_seed(0)
    M, N, K = 64, 64, 256
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-30, 31, (M, 1), generator=g).float())
    w = torch.randn(N, K, generator=g) * torch.exp2(torch.randint(-30, 31, (N, 1), generator=g).float())
    x[:, 128:] = -x[:, :128] * (1 + 2.0 ** -20)
    w[:, 128:] = w[:, :128]
    y = _F().linear_act(x.to(dev), w.to(dev))
    want = x.double() @ w.double().t()
    _within(y, want, _sum_err(K, torch.float32) * (x.double().abs() @ w.double().abs().t()))
    one = torch.eye(64) * 1.2345678           # a single product per sum
    w = w[:, :64].contiguous()
    _within(F_one(one.to(dev), w.to(dev)), one.double() @ w.double().t(), 4 * U * (one.double() @ w.double().abs().t()))


def F_one(x, w):
    return _F().linear_act(x, w)


@pytest.mark.parametrize("dtype", FLOATS)
def test_strided_operands(dev, dtype):
    """Rows a distance apart, a transposed weight, x and residual with more axes."""
    F_ = _F()
    x, w, b, r, dy = _case(24, 40, 32, dtype, 3, True, True)
    base = F_.linear_act(*(t.to(dev) for t in (x, w, b)), "tanh", r.to(dev))
    wide = torch.zeros(24, 50, dtype=dtype)
    wide[:, 9:41] = x
    rw = torch.zeros(24, 64, dtype=dtype)
    rw[:, 8:48] = r
    assert torch.equal(F_.linear_act(wide.to(dev)[:, 9:41], w.to(dev), b.to(dev), "tanh", rw.to(dev)[:, 8:48]), base)
    assert torch.equal(F_.linear_act(x.to(dev), w.t().contiguous().to(dev).t(), b.to(dev), "tanh", r.to(dev)), base)
    assert torch.equal(F_.linear_act(x.view(2, 3, 4, 32).to(dev), w.to(dev), b.to(dev), "tanh", r.view(2, 3, 4, 40).to(dev)),
                       base.view(2, 3, 4, 40))
    xt = x.t().contiguous().to(dev).t()                       # column-major x
    assert torch.equal(F_.linear_act(xt, w.to(dev), b.to(dev), "tanh", r.to(dev)), base)
    one = F_.linear_act(x[0].to(dev), w.to(dev), b.to(dev), "tanh", r[0].to(dev))
    assert one.shape == (40,)
    _within(one, base[0].double().cpu(), 4 * _half(dtype) * base[0].double().cpu().abs() + 1e-6)
    # gradients through views, an expanded dy, and a frozen weight
    big = wide.to(dev).requires_grad_(True)
    F_.linear_act(big[:, 9:41], w.to(dev), b.to(dev), "tanh").sum().backward()
    assert bool((big.grad[:, :9] == 0).all()) and bool((big.grad[:, 41:] == 0).all()) and float(big.grad.abs().sum()) > 0


@pytest.mark.parametrize("dtype", FLOATS)
def test_empty_axes(dev, dtype):
    F_ = _F()
    b = torch.arange(5, dtype=dtype, device=dev).requires_grad_(True)
    y = F_.linear_act(torch.empty(3, 0, dtype=dtype, device=dev), torch.empty(5, 0, dtype=dtype, device=dev), b, "relu")
    assert torch.equal(y, b.detach().expand(3, 5))
    y.sum().backward()
    assert torch.equal(b.grad.cpu(), torch.tensor([0, 3, 3, 3, 3], dtype=dtype))
    x = torch.empty(0, 4, dtype=dtype, device=dev, requires_grad=True)
    w = torch.ones(5, 4, dtype=dtype, device=dev, requires_grad=True)
    b.grad = None
    y = F_.linear_act(x, w, b, "gelu")
    y.sum().backward()
    assert y.shape == (0, 5) and x.grad.shape == (0, 4) and bool((w.grad == 0).all()) and bool((b.grad == 0).all())
    assert F_.linear_act(torch.ones(2, 4, dtype=dtype, device=dev), w.detach()[:0]).shape == (2, 0)


def test_nan_stays_in_its_rows(dev):
    for dtype in FLOATS:
        x, w, b, _, _ = _case(40, 72, 64, dtype, 3)
        clean = _F().linear_act(x.to(dev), w.to(dev), b.to(dev), "relu")
        x[7, 3] = float("nan")
        x[9, 0] = float("inf")
        y = _F().linear_act(x.to(dev), w.to(dev), b.to(dev), "relu")
        keep = [i for i in range(40) if i not in (7, 9)]
        assert torch.equal(y[keep], clean[keep]) and bool(y[7].isnan().all())


def test_neighbouring_memory_is_left_alone(dev):
    """Rows behind the last one, and what lies between the rows of strided inputs (NaN there)."""
    for dtype in FLOATS:
        for M, N, K in ((5, 72, 64), (5, 70, 61)):
            x, w, b, _, _ = _case(M, N, K, dtype, 3)
            xb = torch.full((M + 4, K + 8), float("nan"), dtype=dtype, device=dev)
            xb[:M, :K] = x.to(dev)
            wb = torch.full((N + 4, K + 8), float("nan"), dtype=dtype, device=dev)
            wb[:N, :K] = w.to(dev)
            y = _F().linear_act(xb[:M, :K], wb[:N, :K], b.to(dev), "gelu")
            assert bool(y.isfinite().all())
            base = _F().linear_act(x.to(dev), w.to(dev), b.to(dev), "gelu")
            _within(y, base.double().cpu(), 4 * _half(dtype) * base.double().cpu().abs() + 1e-5)


def test_more_than_2_to_the_31_elements(dev):
    """x and dx of 70000 x 32768 bf16: rows and gradients far behind the first 2^31 elements."""
    M, N, K = 70000, 16, 32768
    x = torch.empty(M, K, dtype=torch.bfloat16, device=dev)
    for i in range(0, M, 10000):
        x[i:i + 10000] = torch.randn(min(10000, M - i), K, device=dev, generator=torch.Generator(dev).manual_seed(i))
    w = (torch.randn(N, K, generator=torch.Generator().manual_seed(1)) / 181).bfloat16().to(dev)
    dy = torch.randn(M, N, generator=torch.Generator().manual_seed(2)).bfloat16().to(dev)
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    y = _F().linear_act(xl, wl)
    dx, dw = torch.autograd.grad(y, [xl, wl], dy)
    rows = torch.tensor([0, 1, 65535, 65536, 65537, M - 2, M - 1], device=dev)
    xs, ws, ds = x.detach()[rows].double(), w.detach().double(), dy[rows].double()
    want = xs @ ws.t().contiguous()
    _within(y.detach()[rows], want.cpu(), (_sum_err(K, torch.bfloat16) * (xs.abs() @ ws.abs().t().contiguous()) + 2.0 ** -8 * want.abs()).cpu())
    want = ds @ ws
    _within(dx[rows], want.cpu(), (_sum_err(N, torch.bfloat16) * (ds.abs() @ ws.abs()) + 2.0 ** -8 * want.abs()).cpu())
    want = mag = 0.0
    for i in range(0, M, 10000):
        a, b = dy[i:i + 10000].double().t().contiguous(), x.detach()[i:i + 10000].double()
        want, mag = want + a @ b, mag + a.abs() @ b.abs()
    _within(dw, want.cpu(), (_sum_err(M, torch.bfloat16) * mag + 2.0 ** -8 * want.abs()).cpu())


def test_tiny_matrices_at_the_end_of_their_memory(dev):
    """Widths below one vector: what is read behind a row must still be the tensor's (the values there are NaN)."""
    for dtype in FLOATS:
        for M, N, K in ((5, 3, 1), (9, 2, 3), (70, 5, 7), (6, 70, 2)):
            x, w, b, _, dy = _case(M, N, K, dtype, 4)
            xb = torch.full((M * K + 64,), float("nan"), dtype=dtype, device=dev)
            xb[:M * K] = x.reshape(-1).to(dev)
            wb = torch.full((N * K + 64,), float("nan"), dtype=dtype, device=dev)
            wb[:N * K] = w.reshape(-1).to(dev)
            _check(dev, xb[:M * K].view(M, K).cpu(), wb[:N * K].view(N, K).cpu(), b, None, dy, "silu", dtype)
            xv, wv = xb[:M * K].view(M, K).requires_grad_(True), wb[:N * K].view(N, K).requires_grad_(True)
            y = _F().linear_act(xv, wv, b.to(dev), "silu")
            grads = torch.autograd.grad(y, [xv, wv], dy.to(dev))
            assert all(bool(t.isfinite().all()) for t in (y, *grads))


def test_no_second_derivative(dev):
    x = torch.randn(3, 4, device=dev, requires_grad=True)
    w = torch.randn(5, 4, device=dev, requires_grad=True)
    (dx,) = torch.autograd.grad(_F().linear_act(x, w, None, "silu").sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", FLOATS)
def test_captured_streams_and_repeats(dev, dtype):
    from lvmhelpers import graphs
    F_ = _F()
    x, w, b, r, dy = (t.to(dev) for t in _case(300, 200, 1200, dtype, 3, True, True))
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    held = {}

    def step():
        y = F_.linear_act(x, w, b, "gelu", r)
        held["out"] = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, _ = graphs.capture(step)
    out = held["out"]
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(300, 1200, generator=torch.Generator().manual_seed(k)).to(dtype))
        graph.replay()
        torch.randn(99, device=dev).sum().item()
        step()
        assert all(torch.equal(p, q) for p, q in zip(out, held["out"]))


def test_modules_are_drop_ins(dev):
    """fuse_linears keeps parameters and state_dict keys, takes activations in, and leaves what it cannot."""
    from lvmhelpers import fused
    torch.manual_seed(0)
    def make():
        return torch.nn.Sequential(torch.nn.Linear(20, 48), torch.nn.ReLU(), torch.nn.Linear(48, 30), torch.nn.GELU(approximate="tanh"),
                                   torch.nn.Sequential(torch.nn.Linear(30, 7, bias=False), torch.nn.Sigmoid()))
    plain = make()
    net = make()
    net.load_state_dict(plain.state_dict())
    params = list(net.parameters())
    assert fused.fuse_linears(net) is net
    assert [n for n, _ in net.named_parameters()] == [n for n, _ in plain.named_parameters()]
    assert all(p is q for p, q in zip(params, net.parameters()))
    assert net[0].activation == "relu" and net[2].activation == "none" and isinstance(net[3], torch.nn.GELU)
    assert net[4][0].activation == "sigmoid" and net[4][0].bias is None and "sigmoid" in repr(net)
    plain, net = plain.to(dev).double(), net.to(dev)
    x = torch.randn(9, 20)
    want = plain(x.to(dev).double())
    got = net(x.to(dev))
    assert float((got.double() - want).abs().max()) <= 200 * U
    want.sum().backward()
    got.sum().backward()
    for p, q in zip(plain.parameters(), net.parameters()):
        assert float((p.grad - q.grad.double()).abs().max()) <= 2000 * U * (1 + float(p.grad.abs().max()))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M", [1, 33, 65, 1000, 70001])
def test_bias_gradient_without_input_features(dev, M, dtype):
    """dy is small whole numbers, at most 4: sums up to 2^18 < 2^24 are exact in fp32 in any order and rounded once
    (in fp16 to infinity from 65520 on, which 2 M does not reach: dy averages to 0)."""
    for act in ("none", "relu"):
        for N in (1, 5, 72):
            dy = torch.randint(-4, 5, (M, N), generator=torch.Generator().manual_seed(M + N)).to(dtype)
            b = torch.ones(N, dtype=dtype, device=dev, requires_grad=True)
            y = _F().linear_act(torch.empty(M, 0, dtype=dtype, device=dev), torch.empty(N, 0, dtype=dtype, device=dev), b, act)
            assert torch.equal(y, torch.ones(M, N, dtype=dtype, device=dev))
            (db,) = torch.autograd.grad(y, [b], dy.to(dev))
            assert torch.equal(db.cpu(), dy.double().sum(0).float().to(dtype))


def _check_tiny_relu(dev, dtype, M, N, K, res):
    """h is a single product, some 2^-27 (below half of fp16's smallest number) of either sign: its slope is 0 or 1.  dy is
    small whole numbers, so db is exact up to its rounding; dx and dw as in _check, dh being exact."""
    g = torch.Generator().manual_seed(M + N)

    def sized(shape, low):                          # +- [1, 1.4) low
        return ((1 + 0.4 * torch.rand(shape, generator=g)) * low * (1 - 2 * torch.randint(0, 2, shape, generator=g))).to(dtype)
    x = torch.zeros(M, K, dtype=dtype)
    at = torch.randint(0, K, (M,), generator=g)
    x[torch.arange(M), at] = sized((M,), 2.0 ** -13)
    w, dy = sized((N, K), 2.0 ** -14), torch.randint(-4, 5, (M, N), generator=g).to(dtype)
    b = torch.zeros(N, dtype=dtype)
    r = torch.randn(M, N, generator=g).to(dtype) if res else None
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
    y = _F().linear_act(*leaves, "relu", None if r is None else r.to(dev))
    X, W, DY = (t.double().to(dev) for t in (x, w, dy))
    h = X @ W.t().contiguous()
    assert float(h.abs().max()) < 2.0 ** -25 and float(h.abs().min()) > 2.0 ** -28
    want = h.clamp_min(0) + (0 if r is None else r.double().to(dev))
    _within(y.detach(), want.cpu(), (_half(dtype) * 1.01 * want.abs() + 2.0 ** -25).cpu())
    dh = DY * (h > 0)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(dev))
    assert torch.equal(db.cpu(), dh.sum(0).to(dtype).cpu())
    _within(dx, (dh @ W).cpu(), (_sum_err(N, dtype) * (dh.abs() @ W.abs()) + _half(dtype) * 1.01 * (dh @ W).abs() + 2.0 ** -25 * (dtype == torch.float16)).cpu())
    dht = dh.t().contiguous()
    _within(dw, (dht @ X).cpu(), (_sum_err(M, dtype) * (dht.abs() @ X.abs()) + _half(dtype) * 1.01 * (dht @ X).abs() + 2.0 ** -25 * (dtype == torch.float16)).cpu())


TINY = [(3, 40, 16), (70, 97, 47), (128, 256, 64), (6, 64, 40000)]      # few rows, unaligned, aligned, split over k


@pytest.mark.parametrize("M,N,K", TINY)
def test_relu_with_a_residual_keeps_the_sign_of_tiny_arguments(dev, M, N, K):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check_tiny_relu(dev, dtype, M, N, K, True)


@pytest.mark.parametrize("M,N,K", TINY)
def test_relu_without_a_residual_keeps_the_sign_of_tiny_arguments(dev, M, N, K):
    """(the sign of y would not do in fp16, where these results are 0)"""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check_tiny_relu(dev, dtype, M, N, K, False)


def test_forward_mode_derivatives_are_refused(dev):
    """Through every public way in; a tensor of the level without a tangent is an ordinary one."""
    import torch.autograd.forward_ad as fwad
    from lvmhelpers import fused
    F_ = _F()
    x, w, z = torch.randn(3, 4, device=dev), torch.randn(5, 4, device=dev), torch.randn(2, 3, device=dev)
    a, v = torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(2, device=dev)
    base, layer = F_.linear_act(x, w), fused.LinearAct(4, 5).to(dev)
    with fwad.dual_level():
        dual, dz = fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(z, torch.ones_like(z))
        for call in (lambda: F_.linear_act(dual, w), lambda: F_.linear_act(dual.view(1, 3, 4), w), lambda: layer(dual),
                     lambda: F_.linear_act(w, dual), lambda: F_.token_logprobs(dz, a), lambda: F_.clipped_policy_loss(dz, a, v, v)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(F_.linear_act(x, w), base)


def test_fp32_products_one_by_one(dev):
    """Single products of any operands, the worst ones of a split in three parts among them (both far from their first
    part's 8 bits).  Left out: 2^-22 |x||w|; rounded: the last sum by u, those before it, of 2^-6 |x||w|
    and less, by less than u in all -- 6 u."""
    g = torch.Generator().manual_seed(0)
    worst = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -7 - 2.0 ** -16, 1 + 2.0 ** -7 - 2.0 ** -15 + 2.0 ** -16 - 2.0 ** -23,
                          1 + 2.0 ** -8 + 2.0 ** -16 - 2.0 ** -23, 1 + 2.0 ** -8, 1 + 2.0 ** -8 - 2.0 ** -23, 2 - 2.0 ** -23, 1.0])
    worst = torch.cat([worst, -worst])
    for M, N in ((64, 64), (256, 512)):
        x, w = 1 + torch.rand(M, generator=g), 1 + torch.rand(N, generator=g)
        x[:16], w[:16] = worst, worst
        x, w = (t * torch.exp2(torch.randint(-30, 31, t.shape, generator=g).float()) for t in (x, w))
        wide = torch.zeros(N, M)                       # row n holds w_n in every column: y[m][n] = x_m w_n
        wide[:] = w[:, None]
        want = x.double()[:, None] * w.double()[None, :]
        _within(F_one(torch.diag(x).to(dev), wide.to(dev)), want, 6 * U * want.abs())


def _slope(name, h):
    phi = 0.5 * torch.erfc(-h * 0.5 ** 0.5)
    s = torch.sigmoid(h)
    return {"none": torch.ones_like(h), "relu": (h > 0).double(), "gelu": phi + h * torch.exp(-0.5 * h * h) / (2 * torch.pi) ** 0.5,
            "silu": s * (1 + h * torch.sigmoid(-h)), "sigmoid": s * torch.sigmoid(-h), "tanh": 1 / torch.cosh(h) ** 2}[name]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_whole_range(dev, act, dtype):
    """Arguments from 0 to the type's largest number, given as the bias (x is 0), so that they are exact; those of bf16 tensors
    are exact in fp16 too, or beyond its range.  Result: 8 u (|a| + 1) and its rounding; slope, summed M times in
    db: M times 12 u, each dh's rounding and the sum's own."""
    big = [65504.0] if dtype == torch.float16 else [65280.0, 1e6, 1e30, 1e38, 3e38]
    h = torch.tensor([0.0, 1e-3, 0.5, 1, 3, 5, 8, 12, 20, 30, 50, 80, 86, 87, 87.5, 88, 88.5, 89, 90, 100, 104, 105, 150, 1000, 1e4] + big)
    h = h.to(dtype)
    assert bool(h.isfinite().all())
    h = torch.cat([h, -h])
    if act == "relu":
        h = h[h != 0]                                   # (the corner has no slope)
    H, N, half = h.double(), h.numel(), _half(dtype)
    for M in (3, 40):
        b = h.to(dev).requires_grad_(True)
        x, w = torch.zeros(M, 8, dtype=dtype, device=dev), torch.ones(N, 8, dtype=dtype, device=dev)
        y = _F().linear_act(x, w, b, act)
        a = 0.5 * H * torch.erfc(-H * 0.5 ** 0.5) if act == "gelu" else _act(act, H)
        want = a.expand(M, N)
        _within(y.detach(), want, 8 * U * (want.abs() + (act not in ("none", "relu"))) + 1.01 * half * want.abs() + 2.0 ** -25 * (dtype == torch.float16))
        (db,) = torch.autograd.grad(y, [b], torch.ones(M, N, dtype=dtype, device=dev))
        s = M * _slope(act, H)
        _within(db, s, M * (12 * U * (act not in ("none", "relu")) + 2.0 ** -25 * (dtype == torch.float16)) + (2.02 * half + 60 * U) * s.abs())


def test_fp32_gelu_keeps_relative_accuracy_in_its_tail(dev):
    """Phi(h) of h < 0 down to fp32's smallest normal numbers.  z = h / sqrt 2 and h^2 / 2 are rounded, which moves Phi and
    e^(-h^2 / 2) by 2 z^2 u = h^2 u and a half of it, relative; erfc is good to 32 u, the rest to 8.  The slope is
    Phi + h phi, each as good."""
    h = -torch.linspace(0.5, 12.5, 2001)
    H = h.double()
    phi, pdf = 0.5 * torch.erfc(-H * 0.5 ** 0.5), torch.exp(-0.5 * H * H) / (2 * torch.pi) ** 0.5
    rel = (2 * H * H + 40) * U
    for M in (3, 40):
        b = h.to(dev).requires_grad_(True)
        y = _F().linear_act(torch.zeros(M, 8, device=dev), torch.ones(h.numel(), 8, device=dev), b, "gelu")
        _within(y.detach(), (H * phi).expand(M, -1), (rel * (H * phi).abs()).expand(M, -1))
        (db,) = torch.autograd.grad(y, [b], torch.ones_like(y))
        _within(db, M * (phi + H * pdf), M * (rel + 40 * U) * (phi + (H * pdf).abs()))
