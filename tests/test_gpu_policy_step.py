"""GPU: the training-step operators together, as a user runs them: a sender network of LinearAct layers, the clipped
policy loss on its symbols, AdamW -- eagerly, in one HIP graph, and next to the same step in torch's fp64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Sender(torch.nn.Module):
    """image features -> logits over symbols, with GraphedStep's calling convention."""

    def __init__(self, feat, hidden, vocab):
        super().__init__()
        self.net = torch.nn.Sequential(torch.nn.Linear(feat, hidden), torch.nn.GELU(), torch.nn.Linear(hidden, hidden),
                                       torch.nn.Tanh(), torch.nn.Linear(hidden, vocab))

    def forward(self, x, symbols, old, adv, ref, mask):
        from lvmhelpers import functional as F_
        loss, stats = F_.clipped_policy_loss(self.net(x), symbols, old, adv, ref, mask, 0.2, 0.3, 0.05, 0.01)
        return {"loss": loss, "log": stats}


def _batch(dev, rows, feat, vocab, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, feat, generator=g).to(dtype)
    symbols = torch.randint(0, vocab, (rows,), generator=g)
    old = -torch.rand(rows, generator=g) * 2 - 4
    adv = torch.randn(rows, generator=g)
    ref = old + torch.randn(rows, generator=g) * 0.2
    mask = torch.rand(rows, generator=g) < 0.8
    return tuple(t.to(dev) for t in (x, symbols, old, adv, ref, mask))


def _reference_step(net, batch):
    """The loss and its gradients, in fp64 by torch's autograd."""
    x, symbols, old, adv, ref, mask = (t.double() if t.is_floating_point() else t for t in batch)
    lsm = torch.log_softmax(net(x), -1)
    logp = lsm.gather(1, symbols[:, None]).squeeze(1)
    ratio = (logp - old).exp()
    surrogate = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.3) * adv)
    d = ref - logp
    per = surrogate + 0.05 * (d.exp() - d - 1) - 0.01 * torch.special.entr(lsm.exp()).sum(1)
    return (per * mask).sum() / mask.sum().clamp_min(1)


@pytest.mark.parametrize("rows,feat,hidden,vocab", [(64, 4096, 256, 256), (33, 77, 129, 1003), (1, 16, 8, 3)])
def test_one_step_against_fp64(dev, rows, feat, hidden, vocab):
    from lvmhelpers import fused, optim
    torch.manual_seed(0)
    model = Sender(feat, hidden, vocab)
    exact = torch.nn.Sequential(*[m for m in Sender(feat, hidden, vocab).net]).double()
    exact.load_state_dict(model.net.state_dict())
    exact = exact.to(dev)
    model = fused.fuse_linears(model).to(dev)
    assert sum(isinstance(m, fused.LinearAct) for m in model.modules()) == 3
    batch = _batch(dev, rows, feat, vocab, 1)
    out = model(*batch)
    out["loss"].backward()
    want = _reference_step(exact, batch)
    want.backward()
    # fp32 through three layers of K <= 4096 products (64 u each at most, as summed here), a softmax and the loss:
    # a relative 2000 u of each gradient's largest entry
    assert abs(float(out["loss"].detach()) - float(want.detach())) <= 2000 * U * max(1.0, abs(float(want.detach())))
    for p, q in zip(model.parameters(), exact.parameters()):
        assert float((p.grad.double() - q.grad).abs().max()) <= 2000 * U * max(float(q.grad.abs().max()), 1e-3)
    # from the same gradients, AdamW moves the weights as torch's does in fp64
    ours = optim.AdamW(model.parameters(), lr=1e-3, weight_decay=0.1)
    theirs = torch.optim.AdamW(exact.parameters(), lr=1e-3, weight_decay=0.1)
    for p, q in zip(model.parameters(), exact.parameters()):
        q.grad = p.grad.double()
    ours.step()
    theirs.step()
    for p, q in zip(model.parameters(), exact.parameters()):
        assert float((p.double() - q).abs().max()) <= 8 * U * float(q.abs().max()) + 40 * U * 1e-3


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graphed_steps_equal_eager_ones(dev, dtype, bits):
    """Several batches through one captured step (forward, backward, optimiser), each against the eager twin: bit for
    bit, for every launch and every sum has a fixed order."""
    from lvmhelpers import fused, optim
    from lvmhelpers.graphs import GraphedStep
    models, opts = [], []
    for _ in range(2):
        torch.manual_seed(0)
        models.append(fused.fuse_linears(Sender(200, 96, 1000)).to(dev).to(dtype))
        opts.append(optim.AdamW(models[-1].parameters(), lr=1e-2, state_bits=bits, min_8bit_size=256))
    step = GraphedStep(models[0], opts[0], _batch(dev, 50, 200, 1000, 0, dtype))
    for k in range(5):
        batch = _batch(dev, 50, 200, 1000, k, dtype)
        out = step(*batch)
        torch.randn(1000, device=dev).sum().item()
        opts[1].zero_grad(set_to_none=True)
        twin = models[1](*batch)
        twin["loss"].backward()
        opts[1].step()
        assert torch.equal(out["loss"].detach(), twin["loss"].detach())
        assert all(torch.equal(p, q) for p, q in zip(models[0].parameters(), models[1].parameters()))
    assert int(opts[0].state[next(models[0].parameters())]["step"]) == 5


def test_two_graphs_of_one_model_side_by_side(dev):
    """Two captures of the loss and its gradients (other batch sizes), replayed in turn and on two streams: neither
    uses the other's workspace."""
    from lvmhelpers import fused, graphs
    torch.manual_seed(0)
    model = fused.fuse_linears(Sender(64, 48, 500)).to(dev)
    params = list(model.parameters())
    runs = []
    for rows in (17, 200):
        batch = _batch(dev, rows, 64, 500, rows)
        held = {}

        def run(batch=batch, held=held):
            out = model(*batch)
            held["out"] = [out["loss"].detach()] + list(torch.autograd.grad(out["loss"], params))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        want = [t.clone() for t in held["out"]]
        held.clear()
        graph, _ = graphs.capture(run)
        runs.append((graph, held["out"], want, batch))          # (a graph reads its batch where it was captured)
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(3):
        for (graph, *_), s in zip(runs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for _, got, want, _ in runs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
