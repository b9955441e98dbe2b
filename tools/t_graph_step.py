"""GPU box: a batch-64 step (cfg5: 1024), eager and captured and replayed N times (also for a rocprofv3 kernel trace of what
a replay is made of):  python tools/t_graph_step.py cfg4|cfg4_topk|cfg1|cfg2|cfg5 [replays] [own]
`own`: the model's layers through fused.fuse_linears and optim.AdamW instead of torch's layers and Adam."""
import sys
import time
import torch
sys.path[:0] = ['.', 'sparse-marginalization-lvm_amd']
import bench_models as bm
from lvmhelpers import fused, optim
from lvmhelpers.graphs import GraphedStep
dev = torch.device('cuda:0')
which = sys.argv[1] if len(sys.argv) > 1 else 'cfg4'
n = int(sys.argv[2]) if len(sys.argv) > 2 else 200
own = 'own' in sys.argv[3:]
if which == 'cfg1':
    m, b = bm.make_ssvae(dev, 64, compact=True)
elif which == 'cfg2':
    m, b = bm.make_signal_game(dev, 64, compact=True, hoist=True)
    m.static_cap = 32
elif which == 'cfg5':
    m, b = bm.make_bitvae(dev, 1024, 128, 'sparsemap')
else:
    m, b = bm.make_bitvae(dev, 64, 32, 'topksparse' if 'topk' in which else 'sparsemap')
if own:
    fused.fuse_linears(m)
    opt = optim.AdamW(m.parameters(), lr=1e-30, weight_decay=0.0)
else:
    opt = torch.optim.Adam(m.parameters(), lr=1e-30, capturable=True)


def timed(step, n):
    for _ in range(10):
        step()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(n):
        step()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) / n * 1e3


tag = f"{which}, {'own layers and AdamW' if own else 'torch layers and Adam'}"
print(f"{tag}: {timed(lambda: bm.train_step(m, opt, b), max(10, n // 4)):.3f} ms per eager step", flush=True)
if which != 'cfg5':     # (static shapes would feed its decoder several times the rows)
    step = GraphedStep(m, opt, b)
    print(f"{tag}: {timed(lambda: step(*b), n):.3f} ms per replayed step, {step.memsets_replaced} memset nodes replaced", flush=True)
