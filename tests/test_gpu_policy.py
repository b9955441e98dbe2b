"""GPU tests of token_logprobs and clipped_policy_loss (csrc/policy.hip) against the formulas in 64 bits.

Tolerances, u = 2^-24.  y = (z - m) log2 e is off by at most 3 u |y| <= 3 u log2 e 2 max|z|; exp2 of it adds 2 u; a sum of V positive terms by
lanes and trees of depth d <= 64 + 20 is off by d u; so log s and logp by
    E = u (6 max|z| + 90)   (3 * 2 * log2 e * ln 2 = 6)
(V <= 140000: a lane adds at most V / 1024 terms in a row, 16 vectors of 8, plus the tree; the bound
uses 150 for those).  The entropy's error is at most the same relative error of p times sum p |log p|
plus E; dz = p (...) inherits 2 E relative, plus half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _F():
    from lvmhelpers import functional
    return functional


def _err(z, V):
    top = z.double().where(z.isfinite(), 0.0).abs().max()
    return U * (6 * float(top) + 90 + min(V, 256) + V / 1024)


def _reference(z, actions, mask=None):
    """fp64 (logp, entropy, p, log p) with 0 where the probability is 0; z any float type, on the CPU."""
    z = z.double()
    lsm = torch.log_softmax(z, -1)
    p = lsm.exp()
    ent = torch.special.entr(p).sum(-1)
    logp = lsm.gather(-1, actions.unsqueeze(-1)).squeeze(-1)
    return logp, ent, p, torch.where(p > 0, lsm, 0.0)


def _grad_reference(p, lsm, ent, actions, c, h):
    dz = -p * (c.unsqueeze(-1) + h.unsqueeze(-1) * (lsm + ent.unsqueeze(-1)))
    return dz.scatter_add_(-1, actions.unsqueeze(-1), c.unsqueeze(-1))


def _logits(shape, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _close(got, want, tol):
    assert got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


# one element to the longest rows: every lane-group size and vector count, and rows that end inside a vector
WIDTHS = [1, 2, 7, 8, 9, 31, 33, 64, 65, 255, 256, 511, 513, 1000, 1023, 2049, 4099, 8191, 10007, 16385, 32003, 40001,
          65537, 66001, 128000, 131073, 140001]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("V", WIDTHS)
def test_logprobs_and_their_gradient_at_every_width(dev, V, dtype):
    rows = 5 if V > 2000 else 37
    z = _logits((rows, V), dtype, V)
    g = torch.Generator().manual_seed(V + 1)
    a = torch.randint(0, V, (rows,), generator=g)
    a[0], a[1] = 0, V - 1
    gl, ge = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    logp, ent, p, lsm = _reference(z, a)
    zd = z.to(dev).requires_grad_(True)
    gotl, gote = _F().token_logprobs(zd, a.to(dev))
    err = _err(z, V)
    _close(gotl.detach(), logp, err + U * logp.abs())
    _close(gote.detach(), ent, 3 * err * (1 + ent) + 2 * U)
    (dz,) = torch.autograd.grad([gotl, gote], [zd], [gl.to(dev), ge.to(dev)])
    want = _grad_reference(p, lsm, ent, a, gl.double(), ge.double())
    half = torch.finfo(dtype).eps / 2
    spread = p * (gl.abs().unsqueeze(-1) + ge.abs().unsqueeze(-1) * (lsm.abs() + ent.unsqueeze(-1) + 1))
    tol = half * want.abs() * (dtype != torch.float32) + 6 * err * spread + 4 * U * want.abs() + (
        torch.finfo(dtype).tiny * half if dtype == torch.float16 else 2.0 ** -126)
    assert dz.dtype == dtype
    _close(dz, want, tol + 4 * U * gl.abs().unsqueeze(-1) * torch.zeros_like(p).scatter_(-1, a.unsqueeze(-1), 1.0))


def _policy_problem(b, t, V, dtype, seed, with_mask=True):
    g = torch.Generator().manual_seed(seed)
    z = _logits((b, t, V), dtype, seed)
    a = torch.randint(0, V, (b, t), generator=g)
    logp = _reference(z, a)[0]
    shift = torch.randn(b, t, generator=g) * 0.3
    for edge in (math.log(0.8), math.log(1.3)):      # (the clip's borders themselves say nothing)
        shift = torch.where((shift - edge).abs() < 1e-3, shift + 3e-3, shift)
    old = (logp - shift).float()
    ref = (logp + torch.randn(b, t, generator=g) * 0.4).float()
    adv = torch.randn(b, t, generator=g)
    mask = torch.rand(b, t, generator=g) < 0.7 if with_mask else None
    return z, a, old, adv, ref, mask


def _policy_reference(z, a, old, adv, ref, mask, low, high, klc, entc, mean):
    logp, ent, p, lsm = _reference(z, a)
    live = torch.ones_like(logp) if mask is None else mask.double()
    norm = 1.0 / max(1.0, float(live.sum())) if mean else 1.0
    A = adv.double()
    ratio = (logp - old.double()).exp()
    clipped = ((A > 0) & (ratio > 1 + high)) | ((A < 0) & (ratio < 1 - low))
    used = torch.where(clipped, torch.where(A > 0, 1 + high, 1 - low), ratio)
    loss = -used * A - entc * ent
    c = torch.where(clipped, 0.0, -A * ratio)
    kl = torch.zeros_like(logp)
    if ref is not None:
        d = ref.double() - logp
        kl = torch.expm1(d) - d
        loss = loss + klc * kl
        c = c - klc * torch.expm1(d)
    c, h = c * norm * live, torch.full_like(c, -entc * norm) * live
    return dict(loss=(loss * live).sum() * norm, logp=logp * live, entropy=ent * live, kl=kl * live,
                clipped=clipped & (live > 0), dz=_grad_reference(p, lsm, ent, a, c, h), p=p, lsm=lsm, ent=ent, c=c, h=h,
                ratio=ratio, live=live, norm=norm)


def _check_policy(loss, stats, dz, r, z, dtype, adv):
    V = z.shape[-1]
    err = _err(z, V)
    _close(stats["logp"], r["logp"], err + U * r["logp"].abs())
    _close(stats["entropy"], r["entropy"], 3 * err * (1 + r["entropy"]) + 2 * U)
    _close(stats["kl"], r["kl"], 2 * err * (1 + r["kl"]) + 2 * U * r["kl"])
    assert torch.equal(stats["clipped"].cpu(), r["clipped"])
    per = r["live"] * (2 * err * r["ratio"] * adv.double().abs() + 4 * err * (1 + r["entropy"]) + 2 * err * (1 + r["kl"]))
    loss = loss.detach()
    assert abs(float(loss) - float(r["loss"])) <= float(per.sum()) * r["norm"] + 2 * U * abs(float(r["loss"]))
    if dz is None:
        return
    half = torch.finfo(dtype).eps / 2
    # c itself is off by the ratio's relative error, 2 err, of its parts
    cerr = (2 * err * r["norm"] * r["live"] * (r["ratio"] * adv.double().abs() + 1 + r["kl"])).unsqueeze(-1)
    spread = r["p"] * (r["c"].abs() + r["h"].abs() * (r["ent"] + 1)).unsqueeze(-1) + r["p"] * r["lsm"].abs() * r["h"].abs().unsqueeze(-1)
    one = 1.0 if dtype != torch.float32 else 0.0
    tol = one * half * r["dz"].abs() * (1 + half) + 6 * err * spread + cerr * (1 + r["p"]) + 4 * U * r["dz"].abs() + (
        torch.finfo(dtype).tiny * half if dtype == torch.float16 else 2.0 ** -126)
    _close(dz, r["dz"], tol)
    assert bool((dz.cpu()[r["live"] == 0] == 0).all())


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("b,t,V,mean,with_mask,with_ref", [
    (64, 1, 256, True, False, True),        # the signal game's sender
    (3, 17, 1000, True, True, True),
    (3, 17, 1001, False, True, False),
    (2, 5, 32003, True, True, True),
    (1, 1, 2, True, False, True),
    (4, 3, 70000, False, False, True),
    (2, 2, 140001, True, True, True),
    (7, 300, 10, True, True, True),
])
def test_policy_loss_follows_the_formula(dev, b, t, V, mean, with_mask, with_ref, dtype):
    z, a, old, adv, ref, mask = _policy_problem(b, t, V, dtype, 7 * V + t, with_mask)
    ref = ref if with_ref else None
    klc = 0.07 if with_ref else 0.0
    to = lambda x: None if x is None else x.to(dev)
    zd = z.to(dev).requires_grad_(True)
    loss, stats = _F().clipped_policy_loss(zd, to(a), to(old), to(adv), to(ref), to(mask), 0.2, 0.3, klc, 0.02,
                                           "mean" if mean else "sum")
    (dz,) = torch.autograd.grad(loss, [zd])
    r = _policy_reference(z, a, old, adv, ref, mask, 0.2, 0.3, klc, 0.02, mean)
    _check_policy(loss, stats, dz, r, z, dtype, adv)
    with torch.no_grad():       # the same values without the gradient
        loss2, stats2 = _F().clipped_policy_loss(zd, to(a), to(old), to(adv), to(ref), to(mask), 0.2, 0.3, klc, 0.02,
                                                 "mean" if mean else "sum")
    assert torch.equal(loss, loss2) and all(torch.equal(stats[k], stats2[k]) for k in stats)


@pytest.mark.parametrize("dtype", FLOATS)
def test_other_incoming_gradients_and_a_second_backward(dev, dtype):
    """loss.backward() hands the forward's buffer on; any other incoming gradient, and a second pass
    over a retained graph, is computed from the logits."""
    z, a, old, adv, ref, mask = _policy_problem(3, 9, 5003, dtype, 3)
    r = _policy_reference(z, a, old, adv, ref, mask, 0.2, 0.3, 0.05, 0.02, False)
    args = [x.to(dev) for x in (a, old, adv, ref, mask)]
    zd = z.to(dev).requires_grad_(True)

    def fresh():
        return _F().clipped_policy_loss(zd, *args, 0.2, 0.3, 0.05, 0.02, "sum")[0]
    (one,) = torch.autograd.grad(fresh(), [zd])
    for g in (-2.5, 1024.0, 1.0):
        loss = fresh()
        scaled = dict(r, dz=r["dz"] * g, c=r["c"] * g, h=r["h"] * g, norm=r["norm"] * abs(g))
        for _ in range(2):
            (dz,) = torch.autograd.grad(loss, [zd], torch.full((), g, device=dev), retain_graph=True)
            err = _err(z, 5003)
            half = torch.finfo(dtype).eps / 2 * (dtype != torch.float32)
            spread = scaled["p"] * (scaled["c"].abs() + scaled["h"].abs() * (scaled["ent"] + 12)).unsqueeze(-1)
            cerr = (2 * err * scaled["norm"] * r["live"] * (r["ratio"] * adv.double().abs() + 1 + r["kl"])).unsqueeze(-1)
            tol = half * scaled["dz"].abs() * (1 + half) + 6 * err * spread + cerr * (1 + r["p"]) + 4 * U * scaled["dz"].abs() + (
                torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2 if dtype == torch.float16 else 2.0 ** -126)
            _close(dz, scaled["dz"], tol)
    loss = fresh()
    (first,) = torch.autograd.grad(loss, [zd], retain_graph=True)
    kept = first.clone()
    torch.autograd.grad(loss, [zd], torch.full((), 3.0, device=dev))
    assert torch.equal(first, kept) and torch.equal(first, one)    # handed over, not written again


def test_fp16_gradients_under_a_loss_scale(dev):
    """The mean over many rows leaves fp16's range; with a loss scale the gradient must come from
    fp32 products with it, not from a stored fp16 one."""
    b, t, V, scale = 64, 32, 1001, 65536.0
    z, a, old, adv, ref, mask = _policy_problem(b, t, V, torch.float16, 5)
    r = _policy_reference(z, a, old, adv, ref, mask, 0.2, 0.3, 0.05, 0.0, True)
    zd = z.to(dev).requires_grad_(True)
    loss, _ = _F().clipped_policy_loss(zd, *(x.to(dev) for x in (a, old, adv, ref, mask)), 0.2, 0.3, 0.05, 0.0)
    (loss * scale).backward()
    want = r["dz"] * scale
    err = _err(z, V)
    tol = want.abs() * 2.0 ** -11 * 1.001 + 2.0 ** -25 + 20 * err * scale * r["norm"] * (1 + r["p"]) * 4
    _close(zd.grad, want, tol)


def test_strided_views_are_read_where_they_lie(dev):
    """A shifted slice of [B, T+1, V+3] logits, transposed leading axes, and 2-D and 4-D shapes."""
    F_ = _F()
    full = _logits((4, 6, 515), torch.bfloat16, 1).to(dev)
    a = torch.randint(0, 512, (4, 5), generator=torch.Generator().manual_seed(2)).to(dev)
    view = full[:, 1:, 2:514]
    base = F_.token_logprobs(view.contiguous(), a)
    for got in (F_.token_logprobs(view, a),
                [x.t() for x in F_.token_logprobs(view.transpose(0, 1), a.t())],
                [x.view(4, 5) for x in F_.token_logprobs(view.contiguous().view(20, 512), a.reshape(20))],
                [x.view(4, 5) for x in F_.token_logprobs(view.contiguous().view(2, 2, 5, 512), a.view(2, 2, 5).to(torch.int32))]):
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    spaced = torch.empty(4, 5, 512, 2, dtype=torch.bfloat16, device=dev)[..., 0].copy_(view)     # last stride 2
    assert torch.equal(F_.token_logprobs(spaced, a)[0], base[0])
    leaf = full.clone().requires_grad_(True)
    sliced = leaf[:, 1:, 2:514]
    logp, ent = F_.token_logprobs(sliced, a)
    (logp.sum() + ent.sum()).backward()
    assert bool((leaf.grad[:, 0] == 0).all()) and bool((leaf.grad[:, :, :2] == 0).all()) and float(leaf.grad.abs().sum()) > 0


def test_offsets_over_32_bits(dev):
    """Rows that start beyond 2^31 elements (a strided view of a 4.3 GB buffer) and a gradient there."""
    V, far = 1000, (1 << 31) + 12345
    buf = torch.empty(far + V, dtype=torch.bfloat16, device=dev)
    rows = torch.as_strided(buf, (2, 1, V), (far, V, 1))
    z = _logits((2, 1, V), torch.bfloat16, 3)
    rows.copy_(z.to(dev))
    a = torch.tensor([[5], [999]])
    logp, ent, _, _ = _reference(z, a)
    got = _F().token_logprobs(rows, a.to(dev))
    err = _err(z, V)
    _close(got[0], logp, err + U * logp.abs())
    _close(got[1], ent, 3 * err * (1 + ent) + 2 * U)


def test_infinities_nan_and_bad_actions(dev):
    F_ = _F()
    inf, nan = math.inf, math.nan
    z = torch.randn(10, 300, generator=torch.Generator().manual_seed(0))
    z[0, 100:] = -inf                    # masked-out actions
    z[1] = -inf                          # nothing left
    z[2, 7] = nan
    z[3, 9] = inf
    z[4, :299] = -inf                    # a single action left
    z[5] = torch.finfo(torch.float32).min     # fp32's lowest value: a uniform row; in bf16 it rounds to -inf
    a = torch.tensor([5, 5, 5, 5, 299, 7, -1, 300, 2 ** 40, 11])
    for dtype in (torch.float32, torch.bfloat16):
        zz = z.to(dtype)
        lowest = torch.full((2, 300), torch.finfo(dtype).min, dtype=dtype)      # each type's own lowest value:
        lowest[1, 3] = 0.5                                                      # uniform, and as a mask
        low, lent = F_.token_logprobs(lowest.to(dev), torch.tensor([7, 3], device=dev))
        assert abs(float(low[0]) + math.log(300)) <= 8 * U * 6 and abs(float(lent[0]) - math.log(300)) <= 8 * U * 6
        assert float(low[1]) == 0.0 and float(lent[1]) == 0.0
        minus_inf = bool(zz[5, 0] == -inf)
        zd = zz.to(dev).requires_grad_(True)
        logp, ent = F_.token_logprobs(zd, a.to(dev))
        bad = torch.tensor([0, 1, 1, 1, 0, minus_inf, 1, 1, 1, 0], dtype=torch.bool)
        assert torch.equal(logp.isnan().cpu(), bad)
        assert torch.equal(ent.isnan().cpu(), torch.tensor([0, 1, 1, 1, 0, minus_inf, 0, 0, 0, 0], dtype=torch.bool))
        ok = [0, 4, 9]
        ref = _reference(zz[ok], a[ok])
        err = _err(zz[ok], 300)
        _close(logp.detach()[ok], ref[0], err + U * ref[0].abs())
        _close(ent.detach()[ok], ref[1], 3 * err * (1 + ref[1]) + 2 * U)
        assert float(logp[4]) == 0.0 and float(ent[4]) == 0.0
        if not minus_inf:
            assert abs(float(logp[5]) + math.log(300)) <= 8 * U * 6 and abs(float(ent[5]) - math.log(300)) <= 8 * U * 6
        (dz,) = torch.autograd.grad([logp, ent], [zd], [torch.ones_like(logp), torch.ones_like(ent)])
        assert bool(dz[[0, 4, 9]].isfinite().all()) and bool((dz[0, 100:] == 0).all()) and bool((dz[4] == 0).all())
        assert bool(dz[[1, 2, 3]].isnan().all())
        # behind a mask none of it is read
        mask = ~bad
        f32 = torch.zeros(10, device=dev)
        loss, stats = F_.clipped_policy_loss(zd, a.to(dev), f32, f32 + 1, f32, mask.to(dev), kl_coeff=0.1, entropy_coeff=0.1)
        (dz,) = torch.autograd.grad(loss, [zd])
        assert bool(loss.isfinite()) and bool(dz.isfinite().all()) and bool((dz[bad] == 0).all())
        assert all(bool((stats[k][bad.to(dev)] == 0).all()) for k in stats)


def test_every_row_masked_and_no_rows(dev):
    F_ = _F()
    z = torch.full((3, 4, 50), math.nan, device=dev, requires_grad=True)
    a = torch.zeros(3, 4, dtype=torch.int64, device=dev)
    v = torch.zeros(3, 4, device=dev)
    for red in ("mean", "sum"):
        loss, _ = F_.clipped_policy_loss(z, a, v, v, mask=torch.zeros(3, 4, dtype=torch.bool, device=dev), reduction=red)
        (dz,) = torch.autograd.grad(loss, [z])
        assert float(loss) == 0.0 and bool((dz == 0).all())
        e = torch.empty(0, 4, 50, device=dev, requires_grad=True)
        loss, stats = F_.clipped_policy_loss(e, a[:0], v[:0], v[:0], reduction=red)
        (de,) = torch.autograd.grad(loss, [e])
        assert float(loss) == 0.0 and de.shape == e.shape and stats["logp"].shape == (0, 4)


def test_gradient_against_differences(dev):
    """Central differences of the fp64 reference loss and the kernel's fp32 gradient: the difference
    quotient with step 1e-5 in fp64 is good to 1e-9."""
    z, a, old, adv, ref, mask = _policy_problem(2, 3, 11, torch.float32, 21)
    zd = z.to(dev).requires_grad_(True)
    loss, _ = _F().clipped_policy_loss(zd, *(x.to(dev) for x in (a, old, adv, ref, mask)), 0.2, 0.3, 0.05, 0.1)
    loss.backward()
    for k in range(z.numel()):
        step = torch.zeros(z.numel(), dtype=torch.float64)
        step[k] = 1e-5
        up, down = (_policy_reference(z.double() + s * step.view(z.shape), a, old, adv, ref, mask, 0.2, 0.3, 0.05, 0.1, True)["loss"]
                    for s in (1, -1))
        assert abs(float(zd.grad.reshape(-1)[k]) - float((up - down) / 2e-5)) <= 200 * U


def test_captured_and_replayed(dev):
    """Forward and backward in one capture use the forward's buffer, replay after replay; the forward
    outside (eager) with the backward captured does not."""
    from lvmhelpers import graphs
    F_ = _F()
    b, t, V = 4, 8, 1003
    z = _logits((b, t, V), torch.float32, 1).to(dev).requires_grad_(True)
    a, old, adv, ref, mask = (x.to(dev) for x in _policy_problem(b, t, V, torch.float32, 2)[1:])
    g = torch.ones((), device=dev)
    held = {}

    def step():
        loss, _ = F_.clipped_policy_loss(z, a, old, adv, ref, mask, 0.2, 0.3, 0.05, 0.02)
        held["loss"] = loss.detach()
        (held["dz"],) = torch.autograd.grad(loss, [z], g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, _ = graphs.capture(step)
    out = dict(held)
    for k in range(4):
        with torch.no_grad():
            z.copy_(_logits((b, t, V), torch.float32, 100 + k).to(dev))
            g.fill_([1.0, 3.0, 1.0, -0.5][k])
        graph.replay()
        graph.replay()
        torch.randn(999, device=dev).sum().item()
        step()
        assert torch.equal(out["loss"], held["loss"])
        # g = 1 keeps the fused gradient, other values recompute it from stored fp32 statistics
        assert float((out["dz"] - held["dz"]).abs().max()) == 0.0


def test_two_streams_and_bitwise_repeats(dev):
    z, a, old, adv, ref, mask = (x.to(dev) for x in _policy_problem(8, 40, 2003, torch.bfloat16, 9))
    F_ = _F()

    def run():
        zz = z.detach().requires_grad_(True)
        loss, stats = F_.clipped_policy_loss(zz, a, old, adv, ref, mask, 0.2, 0.3, 0.05, 0.02)
        return [loss.detach(), torch.autograd.grad(loss, [zz])[0]] + list(stats.values())
    first = run()
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(run())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(first, o))


@pytest.mark.parametrize("V,rows", [(200, (1 << 23) + 3), (1500, (1 << 21) + 5)])     # 4 rows and 1 row to a workgroup
def test_rows_of_more_than_two_million_workgroups(V, rows, dev):
    gen = torch.Generator().manual_seed(3)
    z = torch.randn(1, V, generator=gen)
    actions = torch.randint(0, V, (rows,), generator=gen)
    logp, entropy = _F().token_logprobs(z.to(dev).expand(rows, V), actions.to(dev))
    want = torch.log_softmax(z.double()[0], 0)
    # (every row is the same: none may differ; to the formula 64 of fp32's half steps, of which a sum of 1500 terms in
    # a tree, the exponentials and the logarithm take fewer than 40)
    table = torch.full((V,), float("nan"), device=dev)
    table[actions.to(dev)] = logp
    assert torch.equal(table[actions.to(dev)], logp)
    seen = torch.unique(actions)
    assert (table.cpu()[seen].double() - want[seen]).abs().max() <= 2.0 ** -18 * want.abs().max()
    assert torch.equal(entropy, entropy[:1].expand(rows))
    assert abs(float(entropy[0]) + float((want.exp() * want).sum())) <= 2.0 ** -18 * abs(float((want.exp() * want).sum()))
