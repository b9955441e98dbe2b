"""GPU tests of optim.AdamW (csrc/adamw.hip) against the update in 64 bits.

Tolerances of 32-bit states, with u = 2^-24 (half a step of fp32): m is two products and a sum with
rounded constants, 4 u (|b1 m| + |c1 g|); v likewise without cancellation, 6 u v; the quotient
m / (sqrt(v) r + eps) adds at most 12 roundings to m's own error; p two more of p's size.  A 16-bit
p is rounded once more, by half a step of its type.  8-bit states: averages in fp64, rounded once to
fp32, so the codes are the definition's and are compared for equality."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _optim():
    from lvmhelpers import optim
    return optim


def _flat(t):
    """The elements in memory order."""
    return t.as_strided((t.numel(),), (1,), t.storage_offset())


# --------------------------------------------------------------------------- the definition, fp64 on the CPU
def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B9) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(n, seed, step, index):
    key = _mix((_mix((seed + 0x9E3779B9 * step) & 0xFFFFFFFF) + index) & 0xFFFFFFFF)
    return _mix((torch.arange(n, dtype=torch.int64) * 0x9E3779B9 + key) & 0xFFFFFFFF)


TABLE = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()      # 0 ... 448


def _encode(x, u16, floor):
    """x fp64 (values of fp32) -> (codes uint8, scales fp64): of the two e4m3 neighbours of |x| / scale the
    upper one where the distance to the lower, in gaps, plus u reaches 1."""
    n = x.numel()
    pad = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    top = torch.where(pad.isfinite(), pad.abs(), 0.0).amax(1)
    powers = torch.exp2(torch.arange(-100, 121, dtype=torch.float64))
    scale = powers[torch.searchsorted(powers * 448, top)]
    y = (pad.abs() / scale[:, None]).view(-1)[:n]
    safe = torch.where(y.isfinite(), y, 0.0)
    low = (torch.searchsorted(TABLE, safe, right=True) - 1).clamp_max(125)
    code = low + ((safe - TABLE[low]) / (TABLE[low + 1] - TABLE[low]) + u16 / 65536.0 >= 1).long()
    if floor:
        code = torch.where((safe > 0) & (code == 0), 1, code)
    code = torch.where(y.isfinite(), code, 0x7F)
    sign = torch.signbit(x).long() * 0x80
    return (code if floor else code | sign).to(torch.uint8), scale


def _decode(codes, scale):
    return codes.view(torch.float8_e4m3fn).double() * scale.repeat_interleave(256)[:codes.numel()]


class Reference:
    """One parameter's weight and state, flat, in fp64 (8-bit: codes and scales)."""

    def __init__(self, p, bits, index, seed=0, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05):
        self.p, self.bits, self.index, self.seed = _flat(p.detach()).cpu().double(), bits, index, seed
        self.lr, self.betas, self.eps, self.wd, self.t = lr, betas, eps, weight_decay, 0
        n = self.p.numel()
        self.m = self.v = torch.zeros(n, dtype=torch.float64)
        self.codes = [torch.zeros(n, dtype=torch.uint8) for _ in range(2)]
        self.scales = [torch.zeros(-(-n // 256), dtype=torch.float64) for _ in range(2)]

    def step(self, g, dtype):
        b1, b2 = self.betas
        g = g.cpu().double()
        self.t += 1
        if self.bits == 8:
            m0, r0 = (_decode(c, s) for c, s in zip(self.codes, self.scales))
            self.m = (b1 * m0 + (1 - b1) * g).float().double()
            self.v = (b2 * r0 * r0 + (1 - b2) * g * g).float().double()
            u = _random(self.p.numel(), self.seed, self.t, self.index)
            r = self.v.sqrt().float().double()      # (fp32's own root may come from a vector library that rounds otherwise)
            for i, (x, bits, floor) in enumerate(((self.m, u & 0xFFFF, False), (r, u >> 16, True))):
                self.codes[i], self.scales[i] = _encode(x, bits, floor)
            self.mtol = U * self.m.abs()
        else:
            self.mtol = 4 * U * ((b1 * self.m).abs() + ((1 - b1) * g).abs()) + b1 * getattr(self, "mtol", 0.0)
            self.m = b1 * self.m + (1 - b1) * g
            self.v = b2 * self.v + (1 - b2) * g * g
        denom = (self.v / (1 - b2 ** self.t)).sqrt() + self.eps
        size = self.lr / (1 - b1 ** self.t)
        vtol = 6 * U * self.t                      # v's own relative error after t steps
        move = size * self.m / denom
        p = self.p * (1 - self.lr * self.wd) - move
        half = torch.finfo(dtype).eps / 2
        self.ptol = getattr(self, "ptol", 0.0) + 3 * U * self.p.abs() + size * self.mtol / denom + (12 * U + vtol) * move.abs()
        if dtype != torch.float32:
            self.ptol = self.ptol + half * p.abs() * (1 + half) + torch.finfo(dtype).tiny * half
        self.p = p
        return self

    def check(self, p, st):
        got = _flat(p.detach()).cpu()
        assert int(st["step"]) == self.t
        if self.bits == 8:
            for i, key in enumerate(("exp_avg", "exp_rms")):
                assert torch.equal(st[key + "_scale"].cpu().double(), self.scales[i])
                codes = _flat(st[key]).cpu().view(torch.uint8)
                assert torch.equal(codes, self.codes[i])
        else:
            assert bool(((_flat(st["exp_avg"]).cpu().double() - self.m).abs() <= self.mtol).all())
            v = _flat(st["exp_avg_sq"]).cpu().double()
            assert bool(((v - self.v).abs() <= 6 * U * self.t * self.v + 2.0 ** -149).all())
        off = (got.double() - self.p).abs()
        assert bool((off <= self.ptol).all()), float((off / self.ptol).max())
        # the next step starts from the rounded weight
        self.p, self.ptol = got.double(), 0.0


def _param(shape, dtype, dev, seed, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(dev)


def _grad(shape, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(torch.randn(shape, generator=g) * 1.5 - 4)
    return (torch.randn(shape, generator=g) * spread).to(dtype).to(dev)


SHAPES = [(1,), (7,), (255,), (256,), (257,), (3, 5, 7), (2048,), (2049,), (100, 333), (8191,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("g_dtype", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p_dtype", FLOATS)
def test_three_steps_follow_the_definition(dev, p_dtype, g_dtype, bits):
    gt = g_dtype or p_dtype
    params = [_param(s, p_dtype, dev, 10 + i) for i, s in enumerate(SHAPES)]
    opt = _optim().AdamW(params, lr=1e-2, weight_decay=0.05, state_bits=bits, min_8bit_size=1, seed=99)
    refs = [Reference(p, bits, i, seed=99) for i, p in enumerate(params)]
    for t in range(3):
        grads = [_grad(s, gt, dev, 100 * t + i) for i, s in enumerate(SHAPES)]
        opt.step(grads=grads)
        for p, g, r in zip(params, grads, refs):
            r.step(_flat(g), p_dtype).check(p, opt.state[p])


@pytest.mark.parametrize("bits", [32, 8])
def test_any_dense_memory_order_and_alignment(dev, bits):
    """Transposed and permuted weights (with gradients in that order and in another), and views that
    start in the middle of a flat buffer."""
    flat = _param((5000,), torch.float32, dev, 1)
    params = [_param((33, 70), torch.float32, dev, 2).t(), _param((4, 5, 6, 7), torch.float32, dev, 3).permute(0, 2, 3, 1),
              flat[3:1501], flat[1501:4999].view(2, 1749)]
    order = [[d for d, _ in sorted(enumerate(p.stride()), key=lambda e: -e[1])] for p in params]
    before = flat.clone()
    opt = _optim().AdamW(params, lr=1e-2, weight_decay=0.05, state_bits=bits, min_8bit_size=1)
    refs = [Reference(p, bits, i) for i, p in enumerate(params)]
    for t in range(2):
        grads = []
        for i, p in enumerate(params):
            g = _grad(p.shape, torch.float32, dev, 50 * t + i)          # contiguous
            grads.append(g if t else torch.empty_like(p).copy_(g))      # ... and in p's order
        opt.step(grads=grads)
        for p, g, r, o in zip(params, grads, refs, order):
            in_order = g.permute(o).contiguous().reshape(-1)
            r.step(in_order, torch.float32).check(p, opt.state[p])
    assert torch.equal(flat[:3], before[:3]) and torch.equal(flat[4999:], before[4999:])


@pytest.mark.parametrize("bits,n", [(32, 8_500_001), (8, 16_900_003)])
def test_a_large_tensor_counts_once(dev, bits, n):
    """Over 4096 workgroups (the step is counted by a launch of its own), several passes per workgroup (8 bits)."""
    p = _param((n,), torch.float32, dev, 1)
    opt = _optim().AdamW([p], lr=1e-2, weight_decay=0.05, state_bits=bits, min_8bit_size=1)
    ref = Reference(p, bits, 0)
    for t in range(2):
        g = _grad((n,), torch.float32, dev, t)
        opt.step(grads=[g])
        ref.step(g, torch.float32).check(p, opt.state[p])


def test_more_tensors_than_one_launch_holds_and_missing_gradients(dev):
    """95 tensors of mixed sizes; every third has no gradient at first and starts counting later."""
    sizes = [(1 + 37 * i % 5000,) for i in range(95)]
    params = [torch.nn.Parameter(_param(s, torch.float32, dev, i)) for i, s in enumerate(sizes)]
    opt = _optim().AdamW(params, lr=1e-2, weight_decay=0.05)
    refs = [Reference(p, 32, i) for i, p in enumerate(params)]
    for t in range(2):
        for i, p in enumerate(params):
            p.grad = None if (t == 0 and i % 3 == 0) else _grad(p.shape, torch.float32, dev, 7 * i + t)
        opt.step()
        for i, (p, r) in enumerate(zip(params, refs)):
            if p.grad is not None:
                r.step(_flat(p.grad), torch.float32).check(p, opt.state[p])
    assert int(opt._tickets[dev]) == 0
    assert int(opt.state[params[0]]["step"]) == 1 and int(opt.state[params[1]]["step"]) == 2


def test_agrees_with_torch(dev):
    a = [_param(s, torch.float32, dev, i) for i, s in enumerate([(300, 77), (77,), (12345,)])]
    b = [torch.nn.Parameter(p.clone()) for p in a]
    ours = _optim().AdamW(a, lr=3e-3, weight_decay=0.1, betas=(0.8, 0.95), eps=1e-6)
    theirs = torch.optim.AdamW(b, lr=3e-3, weight_decay=0.1, betas=(0.8, 0.95), eps=1e-6)
    for t in range(5):
        grads = [_grad(p.shape, torch.float32, dev, 31 * t + i) for i, p in enumerate(a)]
        for q, g in zip(b, grads):
            q.grad = g.clone()
        ours.step(grads=grads)
        theirs.step()
    for p, q in zip(a, b):   # (5 steps of two fp32 evaluations: 5 * (2 * 3 u |p| + 2 * 30 u lr) with |p| < 1, |move| < 2 lr)
        assert float((p - q.detach()).abs().max()) <= 5 * (6 * U + 120 * U * 3e-3)


def test_zero_and_nonfinite_gradients(dev):
    """An all-zero block decodes to zeros; an infinite or NaN gradient spoils its own element and no
    other one of its 256-element block."""
    for bits in (32, 8):
        p = _param((1024,), torch.float32, dev, 5)
        opt = _optim().AdamW([p], lr=1e-2, state_bits=bits, min_8bit_size=1)
        g = _grad((1024,), torch.float32, dev, 6)
        g[256:512] = 0.0
        opt.step(grads=[g])
        m, v = opt.averages(p)
        assert bool((m[256:512] == 0).all()) and bool((v[256:512] == 0).all()) and bool(p.isfinite().all())
        g = g.clone()
        g[600], g[601] = math.inf, math.nan
        opt.step(grads=[g])
        opt.step(grads=[torch.zeros_like(g)])
        bad = torch.zeros(1024, dtype=torch.bool, device=dev)
        bad[600] = bad[601] = True
        assert bool(p[~bad].isfinite().all()) and bool((~p[bad].isfinite()).all())
        m, _ = opt.averages(p)
        assert bool(m[~bad].isfinite().all()) and bool((~m[bad].isfinite()).all())


def test_tiny_and_huge_values_keep_their_scales(dev):
    """Magnitudes from 1e-38 to 1e18 in one tensor, block by block."""
    mag = torch.logspace(-38, 18, 57).repeat_interleave(256)
    g = (torch.randn(mag.numel(), generator=torch.Generator().manual_seed(1)) * mag).float()
    p = _param((g.numel(),), torch.float32, dev, 5)
    opt = _optim().AdamW([p], lr=1e-2, weight_decay=0.05, state_bits=8, min_8bit_size=1)
    ref = Reference(p, 8, 0)
    gd = g.to(dev)
    for _ in range(2):
        opt.step(grads=[gd])
        ref.step(g, torch.float32)
        st = opt.state[p]
        for i, key in enumerate(("exp_avg", "exp_rms")):
            assert torch.equal(st[key + "_scale"].cpu().double(), ref.scales[i])
            assert torch.equal(st[key].cpu().view(torch.uint8), ref.codes[i])
        assert bool(p.isfinite().all())


def test_stochastic_rounding_moves_the_second_average_as_it_should(dev):
    """Gradients fall to zero: after k steps v has decayed to beta2^k of itself.  Rounded to nearest it
    would not move at all (a step changes r by 0.05 %, codes lie 6 to 12 % apart).  Mean over n
    elements of r_k / r_0: E = prod of the per-step expectations = beta2^(k/2) (rounding is unbiased
    for r; the square root is the same for every element of the step up to the floor of one code);
    the spread of one element after k steps is at most sqrt(k q (1 - beta2) / 2) with q = 1/8, so the
    mean of n = 65536 elements lies within 6 standard errors."""
    n, k, b2 = 65536, 200, 0.999
    p = torch.zeros(n, device=dev)
    opt = _optim().AdamW([p], lr=0.0, betas=(0.9, b2), state_bits=8, min_8bit_size=1, weight_decay=0.0)
    g = torch.ones(n, device=dev)
    opt.step(grads=[g])
    r0 = opt.averages(p)[1].sqrt().mean()
    zero = torch.zeros_like(g)
    for _ in range(k):
        opt.step(grads=[zero])
    ratio = float(opt.averages(p)[1].sqrt().mean() / r0)
    sigma = math.sqrt(k * 0.125 * (1 - b2) / 2)
    assert abs(ratio - b2 ** (k / 2)) <= 6 * sigma / math.sqrt(n)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(dev, bits):
    """A captured step, replayed with eager work between the replays, against an eager twin; the rate
    is a tensor that a schedule changes."""
    from lvmhelpers import graphs
    shapes = [(300, 40), (40,), (5000,)]
    a = [_param(s, torch.float32, dev, i) for i, s in enumerate(shapes)]
    b = [p.clone() for p in a]
    lr_a, lr_b = torch.full((), 1e-2, device=dev), torch.full((), 1e-2, device=dev)
    opt_a = _optim().AdamW(a, lr=lr_a, state_bits=bits, min_8bit_size=1, seed=3)
    opt_b = _optim().AdamW(b, lr=lr_b, state_bits=bits, min_8bit_size=1, seed=3)
    grads = [_grad(s, torch.float32, dev, i) for i, s in enumerate(shapes)]
    for opt in (opt_a, opt_b):
        opt.step(grads=grads)                  # makes the states
    graph, _ = graphs.capture(lambda: opt_a.step(grads=grads))
    for t in range(5):
        for i, g in enumerate(grads):
            g.copy_(_grad(g.shape, torch.float32, dev, 1000 * t + i))
        for lr in (lr_a, lr_b):
            lr.fill_(1e-2 / (t + 1))
        graph.replay()
        torch.randn(1000, device=dev).sum().item()
        opt_b.step(grads=grads)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert all(torch.equal(opt_a.state[p][k].float(), opt_b.state[q][k].float()) for k in opt_a.state[p])
    assert int(opt_a.state[a[0]]["step"]) == 6


def test_another_stream_and_repeatability(dev):
    outs = []
    for _ in range(2):
        p = _param((50000,), torch.bfloat16, dev, 1)
        opt = _optim().AdamW([p], lr=1e-2, state_bits=8, seed=7)
        g = _grad((50000,), torch.bfloat16, dev, 2)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                opt.step(grads=[g])
        torch.cuda.current_stream().wait_stream(side)
        outs.append((p, opt.state[p]["exp_rms"].float()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip_keeps_types_and_addresses(dev, bits):
    p = _param((100, 90), torch.bfloat16, dev, 1)
    opt = _optim().AdamW([p], lr=1e-2, state_bits=bits, min_8bit_size=1)
    gs = [_grad(p.shape, torch.bfloat16, dev, i) for i in range(3)]
    opt.step(grads=[gs[0]])
    saved, weight = opt.state_dict(), p.clone()
    saved = {"param_groups": saved["param_groups"], "state": {k: {n: v.clone() for n, v in s.items()}
                                                              for k, s in saved["state"].items()}}
    opt.step(grads=[gs[1]])
    ptrs = {k: v.data_ptr() for k, v in opt.state[p].items()}
    after = p.clone()
    p.copy_(weight)
    opt.load_state_dict(saved)
    assert {k: v.data_ptr() for k, v in opt.state[p].items()} == ptrs
    opt.step(grads=[gs[1]])
    assert torch.equal(p, after)
    q = weight.clone()
    other = _optim().AdamW([q], lr=1e-2, state_bits=bits, min_8bit_size=1)
    other.load_state_dict(saved)
    other.step(grads=[gs[1]])
    assert torch.equal(q, after) and other.state[q]["exp_avg"].dtype == opt.state[p]["exp_avg"].dtype


def test_replaced_weights_and_states_are_seen(dev):
    """A weight whose storage, and a state whose tensors were exchanged between two steps (weights moved, states
    restored by hand); a parameter resized behind the optimiser's back is refused."""
    p = torch.nn.Parameter(_param((64, 64), torch.float32, dev, 1))
    opt = _optim().AdamW([p], lr=1e-2, weight_decay=0.05)
    ref = Reference(p, 32, 0)
    for t in range(4):
        p.grad = _grad((64, 64), torch.float32, dev, t)
        opt.step()
        ref.step(_flat(p.grad), torch.float32).check(p, opt.state[p])
        if t == 1:
            p.data = p.data.clone()
        if t == 2:
            opt.state[p] = {k: v.clone() for k, v in opt.state[p].items()}
    on_gpu = p.data
    p.data = on_gpu.cpu()                       # (the state stays behind; the gradient goes with it)
    p.grad = torch.zeros(64, 64)
    with pytest.raises(RuntimeError):
        opt.step()
    p.grad = None
    p.data = torch.zeros(64, 65, device=dev)
    p.grad = torch.zeros(64, 65, device=dev)
    with pytest.raises(ValueError):
        opt.step()
    q = torch.nn.Parameter(torch.zeros(10, 4, device=dev))
    opt = _optim().AdamW([q])
    q.grad = torch.sparse_coo_tensor(torch.tensor([[1]], device=dev), torch.ones(1, 4, device=dev), (10, 4))
    with pytest.raises(TypeError):
        opt.step()


def test_small_parameters_keep_32_bits(dev):
    w, b = _param((64, 64), torch.float32, dev, 1), _param((64,), torch.float32, dev, 2)
    opt = _optim().AdamW([w, b], state_bits=8)
    opt.step(grads=[torch.ones_like(w), torch.ones_like(b)])
    assert "exp_rms" in opt.state[w] and "exp_avg_sq" in opt.state[b]


@pytest.mark.parametrize("bits", [32, 8])
def test_inside_a_graphed_training_step(dev, bits):
    """The optimiser where this framework uses one: GraphedStep of the 32-bit VAE against eager steps."""
    import bench_models
    from lvmhelpers.graphs import GraphedStep
    models, losses = [], []
    for graphed in (False, True):
        torch.manual_seed(0)
        model, batch = bench_models.make_bitvae(dev, batch=16, bits=16, mode='topk')
        opt = _optim().AdamW(model.parameters(), lr=1e-3, state_bits=bits)
        if graphed:
            step = GraphedStep(model, opt, batch)
        out = []
        for _ in range(4):
            res = step(*batch) if graphed else bench_models.train_step(model, opt, batch)
            out.append(float(res['loss'].detach()))
        losses.append(out)
        models.append(model)
    # the graphed step weighs every slot, the eager one the support: the same sums in another order
    assert all(abs(x - y) <= 1e-4 * abs(x) for x, y in zip(*losses))


def test_a_graph_that_kept_a_weight_notices_the_step(dev):
    w = torch.nn.Parameter(torch.ones(8, 8, device=dev))
    opt = _optim().AdamW([w])
    x = torch.ones(4, 8, device=dev, requires_grad=True)
    y = x @ w.t()
    w.grad = torch.ones_like(w)
    before = w._version
    opt.step()
    assert w._version > before
    with pytest.raises(RuntimeError):           # dx = dy w needs the weight of before
        y.sum().backward()


def test_a_refused_gradient_leaves_every_parameter_alone(dev):
    p, q = (torch.nn.Parameter(torch.ones(300, device=dev)) for _ in range(2))
    opt = _optim().AdamW([p, q])
    with pytest.raises(TypeError):
        opt.step(grads=[torch.ones(300, device=dev), torch.ones(301, device=dev)])
    torch.cuda.synchronize()
    assert torch.equal(p, torch.ones_like(p)) and torch.equal(q, torch.ones_like(q))
    opt.step(grads=[torch.ones(300, device=dev), torch.ones(300, device=dev)])
    assert int(opt.state[p]["step"]) == 1 and int(opt.state[q]["step"]) == 1


def test_steps_of_one_optimiser_on_two_streams(dev):
    """Disjoint parameters of one optimiser, updated by two graphs on two streams and then by eager steps on them:
    every step is counted, and the weights are an optimiser's that does one after the other."""
    from lvmhelpers import graphs
    n, k = 40, 20
    a = [_param((3000 + i,), torch.float32, dev, i) for i in range(n)]
    b = [p.clone() for p in a]
    opt_a, opt_b = (_optim().AdamW(p, lr=1e-2, weight_decay=0.05) for p in (a, b))
    grads = [_grad(p.shape, torch.float32, dev, i) for i, p in enumerate(a)]
    halves = [[g if i % 2 == h else None for i, g in enumerate(grads)] for h in range(2)]
    opt_a.step(grads=grads)
    both = [graphs.capture(lambda h=h: opt_a.step(grads=halves[h]))[0] for h in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(k):
        for s, graph in zip(streams, both):
            with torch.cuda.stream(s):
                graph.replay()
    for _ in range(k):
        for s, half in zip(streams, halves):
            with torch.cuda.stream(s):
                opt_a.step(grads=half)
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for _ in range(2 * k + 1):
        opt_b.step(grads=grads)
    for p, q in zip(a, b):
        assert torch.equal(p, q) and int(opt_a.state[p]["step"]) == 2 * k + 1


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_goes_on_after_load_state_dict(dev, bits):
    """Replays after load_state_dict use the loaded states and rate and write no memory that was given back: the words
    allocated after the load keep their values, and weights, states and counters are those of an eager twin."""
    from lvmhelpers import graphs
    shapes = [(300, 40), (40,), (5000,)]

    def make(lr):
        ps = [_param(s, torch.float32, dev, i) for i, s in enumerate(shapes)]
        return ps, _optim().AdamW(ps, lr=lr, state_bits=bits, min_8bit_size=1, seed=3)
    lr_a, lr_b = torch.full((), 1e-2, device=dev), torch.full((), 1e-2, device=dev)
    (a, opt_a), (b, opt_b) = make(lr_a), make(lr_b)
    c, opt_c = make(torch.full((), 3e-3, device=dev))          # what is loaded
    grads = [_grad(s, torch.float32, dev, i) for i, s in enumerate(shapes)]
    for _ in range(3):
        opt_c.step(grads=grads)
    for opt in (opt_a, opt_b):
        opt.step(grads=grads)
    graph, _ = graphs.capture(lambda: opt_a.step(grads=grads))
    graph.replay()
    opt_b.step(grads=grads)
    saved = opt_c.state_dict()
    opt_a.load_state_dict(saved)
    opt_b.load_state_dict(saved)
    words = [torch.full((1,), 7, dtype=torch.int32, device=dev) for _ in range(4096)]
    for t in range(4):
        for lr in (lr_a, lr_b):                                # a schedule goes on with the loaded rate
            lr.mul_(0.5 if t else 1.0)
        graph.replay()
        torch.randn(1000, device=dev).sum().item()
        opt_b.step(grads=grads)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert all(torch.equal(opt_a.state[p][k].float(), opt_b.state[q][k].float()) for k in opt_a.state[p])
    assert int(opt_a.state[a[0]]["step"]) == 3 + 4 and abs(float(lr_a) - 3e-3 / 8) < 1e-9
    assert bool((torch.stack(words) == 7).all())
    # and with a state that holds nothing: the next replay is a fresh optimiser's first step
    fresh, opt_f = make(1e-2)
    for f, p in zip(fresh, a):
        f.copy_(p)
    opt_a.load_state_dict(opt_f.state_dict())
    graph.replay()
    opt_f.step(grads=grads)
    assert all(torch.equal(p, f) for p, f in zip(a, fresh)) and int(opt_a.state[a[1]]["step"]) == 1


def test_a_rate_on_the_cpu_is_not_captured(dev):
    """A replay could not see it change."""
    p, g = _param((300,), torch.float32, dev, 1), _grad((300,), torch.float32, dev, 2)
    opt = _optim().AdamW([p], lr=torch.tensor(1e-2))
    opt.step(grads=[g])                            # eagerly it is read at the call
    other = p.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="tensor lr"):
        with torch.cuda.graph(graph):
            opt.step(grads=[g])
    torch.cuda.synchronize()
    assert torch.equal(p, other) and int(opt.state[p]["step"]) == 1
    opt.step(grads=[g])
    assert int(opt.state[p]["step"]) == 2
