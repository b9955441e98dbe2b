"""AdamW as one launch over all parameters, with its states in 32 or in 8 bits.

No counterpart in the reference, whose scripts use torch's optimisers.  A step of a small model is
launch bound (the batch-64 models of `bench_models.py` have 10 to 20 parameter tensors); here the
whole update of up to 40 tensors is one kernel of csrc/adamw.hip, step counters included, and
nothing is read back, so it runs unchanged inside `lvmhelpers.graphs.GraphedStep`.

    opt = AdamW(model.parameters(), lr=1e-3)
    step = GraphedStep(model, opt, first_batch)

`state_bits=8` keeps both averages as e4m3 codes with one power-of-two scale per 256 elements: 2 B
per weight instead of 8.  They are rounded stochastically.  Rounding to nearest would freeze them:
the second average moves by a 1 - beta2 = 0.001 part of itself per step and neighbouring codes
are 6 to 12 % apart, so the nearest code would always be the old one; rounded stochastically the
expected value moves as it should.  The random bits are a hash of (seed, step, tensor, element):
runs repeat bit for bit.
"""
import torch

from . import _native

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_STATE_32 = ("exp_avg", "exp_avg_sq")
_STATE_8 = ("exp_avg", "exp_avg_scale", "exp_rms", "exp_rms_scale")
BLOCK = 256     # elements that share one scale of an 8-bit state


class AdamW(torch.optim.Optimizer):
    """p <- p (1 - lr wd) - lr m^ / (sqrt(v^) + eps), m^ and v^ the bias-corrected averages of the
    gradient and its square (torch.optim.AdamW's update).

    params: float32, float16 or bfloat16 GPU tensors (dense, any memory order); a 16-bit weight is
        updated in fp32 and rounded to nearest.
    lr: a number, or a float32 tensor of one element on the parameters' device, which a captured
        step then reads at every replay.
    state_bits: 32, or 8 for parameters of at least `min_8bit_size` elements (smaller ones -- biases,
        norms -- keep 32 bits).  The choice is made when a parameter's state is first created.
    seed: of the 8-bit states' rounding.

    State per parameter: `step` (int64 on the device) and `exp_avg`, `exp_avg_sq` (float32), or
    `exp_avg`, `exp_rms` (float8_e4m3fn codes; the latter stand for the square root of the second
    average) with `exp_avg_scale`, `exp_rms_scale` (float32, one per 256 elements in memory order).
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 min_8bit_size=4096, seed=0):
        self._order = {}        # parameter -> its number in the rounding hash
        self._tickets = {}      # device -> the kernel's counter word (zero between steps)
        self._checked = {}      # a parameter's number -> what was found of it and its state (_entry)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size, seed=seed, capturable=True))

    def __setstate__(self, state):      # unpickled or deep-copied
        super().__setstate__(state)
        self._order = {p: i for i, p in enumerate(p for g in self.param_groups for p in g["params"])}
        self._tickets, self._checked = {}, {}

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
        except Exception:
            self.param_groups.pop()
            raise
        for p in group["params"]:
            self._order[p] = len(self._order)

    @staticmethod
    def _check_group(group):
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32:
                raise ValueError("AdamW: a tensor lr must be one float32 element")
        elif not lr >= 0:
            raise ValueError(f"AdamW: invalid lr {lr}")
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError(f"AdamW: invalid betas {(b1, b2)}")
        if not group["eps"] >= 0 or not group["weight_decay"] >= 0:
            raise ValueError("AdamW: eps and weight_decay must not be negative")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {group['state_bits']}")
        for p in group["params"]:
            if p.dtype not in _FLOATS:
                raise TypeError(f"AdamW: parameters are float32, float16 or bfloat16, got {p.dtype}")

    # ------------------------------------------------------------------------------------- state
    def _init_state(self, p, group):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter's first step makes its state, which every replay of this capture would "
                               "make anew; run one step before capturing (GraphedStep does)")
        if torch.empty_like(p).stride() != p.stride():
            raise ValueError("AdamW: a parameter's memory must be dense (no gaps, no overlap)")
        st = {"step": torch.zeros((), dtype=torch.int64, device=p.device)}
        if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
            blocks = -(-p.numel() // BLOCK)
            for key in ("exp_avg", "exp_rms"):
                st[key] = torch.zeros_like(p, dtype=torch.float8_e4m3fn, memory_format=torch.preserve_format)
                st[key + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        else:
            for key in _STATE_32:
                st[key] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        self.state[p].update(st)
        return self.state[p]

    def averages(self, p):
        """(exp_avg, exp_avg_sq) of a parameter as float32 tensors, 8-bit states decoded."""
        st = self.state[p]
        if "exp_rms" not in st:
            return st["exp_avg"], st["exp_avg_sq"]
        out = []
        for key in ("exp_avg", "exp_rms"):
            x = st[key].float()
            flat = x.as_strided((x.numel(),), (1,))                     # memory order
            flat.mul_(st[key + "_scale"].repeat_interleave(BLOCK)[:x.numel()])
            out.append(x)
        return out[0], out[1].square_()

    def load_state_dict(self, state_dict):
        """As the base class, but every state keeps its own type (the base class casts floating
        states to the parameter's) and is copied into the tensors that are there already, which
        a captured step goes on using."""
        held = {p: dict(st) for p, st in self.state.items()}
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for key, value in state_dict["state"].get(i, {}).items():
                if not torch.is_tensor(value):
                    continue
                old = held.get(p, {}).get(key)
                if torch.is_tensor(old) and old.shape == value.shape and old.dtype == value.dtype:
                    self.state[p][key] = old.copy_(value)
                else:
                    new = torch.empty_like(p, dtype=value.dtype) if value.shape == p.shape and key != "step" \
                        else torch.empty(value.shape, dtype=value.dtype, device=p.device)
                    self.state[p][key] = new.copy_(value)

    # -------------------------------------------------------------------------------------- step
    @torch.no_grad()
    def step(self, closure=None, *, grads=None):
        """One update.  grads: the gradients to use instead of `.grad`, one entry (or None: the
        parameter is left alone) per parameter in the order of the groups; they may have another type
        than the weight, such as float32 next to bfloat16."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grads is not None:
            grads = list(grads)
            if len(grads) != sum(len(g["params"]) for g in self.param_groups):
                raise ValueError("AdamW.step: grads must have one entry per parameter")
        at = 0
        for group in self.param_groups:
            launches = {}
            keep = []            # gradients in another memory order, laid out anew: alive until the launch
            for p in group["params"]:
                g = p.grad if grads is None else grads[at]
                at += 1
                if g is None or p.numel() == 0:
                    continue
                key, entry = self._entry(p, g, group, keep, at - 1, grads is not None)
                entries = launches.get(key)
                if entries is None:
                    launches[key] = entries = []
                entries.append(entry)
            for (dev, p_dtype, g_dtype, bits), entries in launches.items():
                lr = group["lr"]
                if isinstance(lr, torch.Tensor) and lr.device != dev:
                    if lr.is_cuda:
                        raise ValueError("AdamW: a tensor lr must be on the parameters' device")
                    lr = float(lr)
                ticket = self._tickets.get(dev)
                if ticket is None:
                    ticket = self._tickets[dev] = torch.zeros(1, dtype=torch.int32, device=dev)
                with _native._on(dev):
                    _native.adamw_step(b"".join(entries), p_dtype, g_dtype, bits, group["betas"], group["eps"], lr,
                                       group["weight_decay"], group["seed"], ticket)
        return loss

    def _entry(self, p, g, group, keep, order, foreign):
        """(launch key, table record) of a parameter.  Addresses are read anew every time; what a check has
        found of the very same tensors (`_checked`) is not checked again: a small model's step is bound
        by these lines."""
        st = self.state[p]
        if "step" not in st:
            self._check(p, g)
            st = self._init_state(p, group)
        m = st["exp_avg"]
        v = st.get("exp_avg_sq")
        bits = 32
        if v is None:
            v, bits = st["exp_rms"], 8
        stride = p.stride()
        known = self._checked.get(order)
        if known is None or known[0] is not p or known[1] is not m or known[2] is not v or known[3] != stride:
            kinds = (torch.float32, torch.float32) if bits == 32 else (torch.float8_e4m3fn, torch.float8_e4m3fn)
            if m.shape != p.shape or v.shape != p.shape or m.stride() != stride or v.stride() != stride:
                raise ValueError("AdamW: a parameter changed its shape or memory order after its state was made")
            if (m.dtype, v.dtype) != kinds or st["step"].dtype != torch.int64:
                raise TypeError("AdamW: a parameter's state has other types than this optimiser made it with")
            self._check(p, g)
            self._checked[order] = known = (p, m, v, stride, p.numel(), self._order[p])
        elif foreign or g.layout != torch.strided:       # (torch itself keeps .grad to its parameter's shape and device)
            self._check(p, g)
        if not (p.is_cuda and g.is_cuda and m.is_cuda and v.is_cuda and st["step"].is_cuda) or p.dtype not in _FLOATS:
            raise _native.NativeError("AdamW: a parameter, its gradient or its state left the GPU, or changed its type")
        if g.stride() != stride:
            g = torch.empty_like(p, dtype=g.dtype).copy_(g)
            keep.append(g)
        if bits == 8:
            blocks = -(-known[4] // BLOCK)
            if any(t.numel() != blocks or t.dtype != torch.float32 or not t.is_cuda
                   for t in (st["exp_avg_scale"], st["exp_rms_scale"])):
                raise ValueError("AdamW: the scales of an 8-bit state do not fit its parameter")
            entry = _native.ADAMW_ENTRY.pack(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(),
                                             st["exp_avg_scale"].data_ptr(), st["exp_rms_scale"].data_ptr(),
                                             st["step"].data_ptr(), known[4], known[5])
        else:
            entry = _native.ADAMW_ENTRY.pack(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), 0, 0,
                                             st["step"].data_ptr(), known[4], known[5])
        return (p.device, p.dtype, g.dtype, bits), entry

    @staticmethod
    def _check(p, g):
        if not p.is_cuda or g.device != p.device:
            raise _native.NativeError("AdamW: parameters and gradients must be on one GPU (there is no CPU fallback)")
        if g.layout != torch.strided or g.dtype not in _FLOATS or g.shape != p.shape:
            raise TypeError(f"AdamW: a gradient must be a dense float32, float16 or bfloat16 tensor of the "
                            f"parameter's shape {tuple(p.shape)}, got {g.dtype} {tuple(g.shape)} ({g.layout})")
