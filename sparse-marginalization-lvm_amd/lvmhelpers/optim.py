"""AdamW as one launch over all parameters, with its states in 32 or in 8 bits.

No counterpart in the reference, whose scripts use torch's optimisers.  A step of a small model is
launch bound (the batch-64 models of `bench_models.py` have 10 to 20 parameter tensors); here the
whole update of up to 40 tensors is one kernel of csrc/adamw.hip, step counters included (captured, and for
large models, they are a second, small one), and nothing is read back, so it runs unchanged inside
`lvmhelpers.graphs.GraphedStep`.

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
BLOCK = 256     # elements that share one scale of an 8-bit state


class AdamW(torch.optim.Optimizer):
    """p <- p (1 - lr wd) - lr m^ / (sqrt(v^) + eps), m^ and v^ the bias-corrected averages of the
    gradient and its square (torch.optim.AdamW's update).

    params: float32, float16 or bfloat16 GPU tensors (dense, any memory order, no two of them sharing
        memory); a 16-bit weight is updated in fp32 and rounded to nearest.
    lr: a number, or a float32 tensor of one element on the parameters' device, which a captured
        step then reads at every replay (one on the CPU is read when a step is called, and refused in a capture).
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
        self._tickets = {}      # device or (device, stream) -> the kernel's counter word (zero between steps)
        self._captured = False  # a graph may hold the addresses of weights, states and rates
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size, seed=seed, capturable=True))

    def __setstate__(self, state):      # unpickled, deep-copied, or from the base class's load_state_dict
        super().__setstate__(state)
        self._order = {p: i for i, p in enumerate(p for g in self.param_groups for p in g["params"])}
        self.__dict__.setdefault("_tickets", {})
        self.__dict__.setdefault("_captured", False)
        if "_loading" in self.__dict__:
            self._load(*self.__dict__.pop("_loading"))

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
        if len(set(map(id, group["params"]))) != len(group["params"]):
            raise ValueError("AdamW: a parameter may be in a group only once")
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
        states to the parameter's), and what a captured step uses stays where it is: values are copied
        into the tensors of the states and of a tensor `lr` that are there already (a number that is loaded
        for a tensor lr fills it).  Once a step has been captured, a state that state_dict does not have
        starts anew in its own memory, and one of another kind (32 for 8 bits) is refused."""
        # (a hook behind the caller's own sees the dict that is loaded; __setstate__ runs before the hooks that follow)
        handle = self.register_load_state_dict_pre_hook(AdamW._before_load)
        try:
            super().load_state_dict(state_dict)
        finally:
            handle.remove()
            self.__dict__.pop("_loading", None)

    def _before_load(self, state_dict):
        held = {p: dict(st) for p, st in self.state.items()}
        rates = [g["lr"] for g in self.param_groups]
        loaded = {p: state_dict["state"].get(i, {}) for g, saved in zip(self.param_groups, state_dict["param_groups"])
                  for i, p in zip(saved["params"], g["params"])}
        if self._captured:
            for p, st in loaded.items():
                if held.get(p) and st and any(not torch.is_tensor(st.get(k)) or st[k].shape != old.shape or st[k].dtype != old.dtype
                                              for k, old in held[p].items()):
                    raise ValueError("AdamW.load_state_dict: a captured step uses a state of another kind; load into a new optimiser")
        first = {}
        for rate, saved in zip(rates, state_dict["param_groups"]):
            if torch.is_tensor(rate) and float(first.setdefault(id(rate), saved["lr"])) != float(saved["lr"]):
                raise ValueError("AdamW.load_state_dict: groups that share one tensor lr would get different rates")
        self._loading = held, rates, loaded

    @torch.no_grad()
    def _load(self, held, rates, loaded):
        for group, rate in zip(self.param_groups, rates):
            if torch.is_tensor(rate):
                rate.copy_(group["lr"]) if torch.is_tensor(group["lr"]) else rate.fill_(group["lr"])
                group["lr"] = rate
        for p, st in loaded.items():
            if self._captured and held.get(p) and not st:
                for old in held[p].values():
                    old.zero_()
                self.state[p] = held[p]
            for key, value in st.items():
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
            params = group["params"]
            if grads is None:
                given = [p.grad for p in params]
            else:
                given = grads[at:at + len(params)]
                at += len(params)
            states = []
            for p, g in zip(params, given):
                if g is None or p.numel() == 0:
                    states.append(None)
                    continue
                st = self.state[p]
                if "step" not in st:
                    if not p.is_cuda:
                        raise _native.NativeError("AdamW: parameters must be on a GPU (there is no CPU fallback)")
                    st = self._init_state(p, group)
                states.append(st)
            if _native.autograd().adamw_step(params, given, states, [self._order[p] for p in params], self._tickets, group["lr"],
                                             *group["betas"], group["eps"], group["weight_decay"], group["seed"] & 0xFFFFFFFF):
                self._captured = True
        return loss
