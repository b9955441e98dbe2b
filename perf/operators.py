"""Measured cases of the training-step operators: `linear_act`, `token_logprobs` /
`clipped_policy_loss` and `optim.AdamW`, each next to its plain form in elementary torch operations.

    own = False     run() computes the plain form, in 32 bits (64 where rounding decisions hang on it)
    own = True      run() makes the calls a user of lvmhelpers makes

A case is a dict of plain values.  `op` is "linear", "policy", "logprobs" or "adamw"."""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_ACTS = ("none", "relu", "gelu", "silu", "sigmoid", "tanh")

# the semi-supervised VAE's 20 parameter tensors: classifier, encoder, decoder
_SSVAE = ("256x784,256,256x256,256,256x256,256,10x256,10,"
          "128x794,128,128x128,128,16x128,16,128x18,128,128x128,128,784x128,784")


def listed():
    return [
        # one token through a square projection with a residual, as served: all weight bytes, no reuse
        {"name": "linear one row", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16",
         "act": "silu", "bias": True, "res": True, "train": False},
        # the bit-vector VAE's output layer over the support rows of 1024 samples: 3920 = 784 pixels x rank 5
        {"name": "linear vae output", "op": "linear", "m": 53000, "n": 3920, "k": 128, "dtype": "f32",
         "act": "none", "bias": True, "res": False, "train": True},
        # nothing divides anything: unaligned rows in every operand
        {"name": "linear ragged", "op": "linear", "m": 1001, "n": 777, "k": 333, "dtype": "f16",
         "act": "gelu", "bias": True, "res": False, "train": True},
        # a feed-forward block's projection over a long batch of tokens
        {"name": "linear long batch", "op": "linear", "m": 8192, "n": 8192, "k": 4096, "dtype": "bf16",
         "act": "gelu", "bias": True, "res": True, "train": True},
        # the signal game's sender as a policy: 64 games, 256 symbols
        {"name": "policy signal game", "op": "policy", "b": 64, "t": 1, "v": 256, "dtype": "f32",
         "reduction": "mean", "pad": 0, "train": True},
        # sequences of many lengths (some empty), the logits a shifted view, a vocabulary that no vector width divides
        {"name": "policy ragged", "op": "policy", "b": 9, "t": 211, "v": 32003, "dtype": "f16",
         "reduction": "sum", "pad": 5, "train": True},
        # a long batch over a large vocabulary
        {"name": "policy long batch", "op": "policy", "b": 8, "t": 1024, "v": 128000, "dtype": "bf16",
         "reduction": "mean", "pad": 0, "train": True},
        # log-probabilities under the policy that acted, for one batch of games and for one of sequences
        {"name": "logprobs signal game", "op": "logprobs", "b": 64, "t": 1, "v": 256, "dtype": "f32",
         "pad": 0, "train": False},
        {"name": "logprobs of a batch", "op": "logprobs", "b": 16, "t": 512, "v": 65536, "dtype": "bf16",
         "pad": 0, "train": False},
        # every parameter of the batch-64 semi-supervised VAE: launch bound
        {"name": "adamw small model", "op": "adamw", "shapes": _SSVAE, "dtype": "f32", "grad": "f32",
         "bits": 32},
        # a large fp32 model
        {"name": "adamw large model", "op": "adamw", "shapes": "8192x8192,8192,8192x8192,8192,16384x8192,"
         "16384,8192x16384,8192", "dtype": "f32", "grad": "f32", "bits": 32},
        # 8-bit states next to bf16 weights, sizes that end inside a block
        {"name": "adamw 8-bit states", "op": "adamw", "shapes": "4099x4097,4099,8191x4097,8191,4097x8191,"
         "4097,32003x1001,1001", "dtype": "bf16", "grad": "bf16", "bits": 8},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "policy", "logprobs", "adamw"])
    if op == "linear":
        while True:
            c = {"op": op, "m": _spread(rng, 1, 53000), "n": _spread(rng, 10, 8192),
                 "k": _spread(rng, 10, 8192), "dtype": rng.choice(["f32", "bf16", "f16"]),
                 "act": rng.choice(_ACTS), "bias": rng.random() < 0.8, "res": rng.random() < 0.4,
                 "train": rng.random() < 0.7}
            if rng.random() < 0.5:   # widths of models are mostly round, numbers of rows never are
                c["n"], c["k"] = max(16, c["n"] // 64 * 64), max(16, c["k"] // 64 * 64)
            if c["m"] * c["n"] * c["k"] <= (1 << (35 if c["dtype"] == "f32" else 37)):
                return c
    if op in ("policy", "logprobs"):
        while True:
            dtype = rng.choice(["f32", "bf16", "f16"])
            c = {"op": op, "b": _spread(rng, 1, 64), "t": _spread(rng, 1, 1024), "v": _spread(rng, 2, 128000),
                 "dtype": dtype, "pad": rng.choice([0, 0, 1, 7]), "train": op == "policy"}
            if op == "policy":   # (a mean over many tokens leaves the range of an fp16 gradient)
                c["reduction"] = "sum" if dtype == "f16" else rng.choice(["mean", "mean", "sum"])
            if c["pad"] + 2 <= c["v"] and c["b"] * c["t"] * c["v"] <= 1 << 29:
                return c
    total = _spread(rng, 1000, 200_000_000)
    shapes = []
    for _ in range(rng.randint(1, 7)):
        part = max(1, int(total * rng.uniform(0.02, 0.3)))
        cols = _spread(rng, 1, 4096)
        rows = max(1, part // cols)
        shapes += ["%dx%d" % (rows, cols), "%d" % rows]
    return {"op": "adamw", "shapes": ",".join(shapes), "dtype": rng.choice(["f32", "bf16", "f16"]),
            "grad": rng.choice(["same", "f32"]), "bits": rng.choice([8, 32])}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _grad_type(case):
    return case["dtype"] if case["grad"] == "same" else case["grad"]


def work(case):
    if case["op"] == "linear":
        m, n, k, e = case["m"], case["n"], case["k"], _SIZE[case["dtype"]]
        b = e * (m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["res"] else 0))
        f = 2.0 * m * n * k
        if case["train"]:   # read dy, write dx, dw, db (dresidual is dy)
            b += e * (m * n + m * k + n * k + (n if case["bias"] else 0))
            f *= 3
        return {"bytes": b, "flops": f}
    if case["op"] in ("policy", "logprobs"):
        rows, v, e = case["b"] * case["t"], case["v"], _SIZE[case["dtype"]]
        b = rows * v * e * (2 if case["train"] else 1) + rows * (8 + 8 + (17 if case["train"] else 0))
        return {"bytes": b, "flops": rows * v * (9.0 if case["train"] else 5.0)}
    n = sum(math.prod(s) for s in _shapes(case))
    per = 2 * _SIZE[case["dtype"]] + _SIZE[_grad_type(case)] + (16 if case["bits"] == 32 else 4 + 16 / 256)
    return {"bytes": n * per, "flops": n * (14.0 if case["bits"] == 32 else 40.0)}


# ------------------------------------------------------------------------------------------ inputs
LR, BETAS, EPS, DECAY, SEED, STEPS_DONE = 1e-3, (0.9, 0.999), 1e-8, 0.01, 1234, 100
CLIP_LOW, CLIP_HIGH, KL, ENT = 0.2, 0.28, 0.05, 0.01


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 17)


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"
    if case["op"] == "linear":
        dt, m, n, k = _DT[case["dtype"]], case["m"], case["n"], case["k"]

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, generator=g, device=dev).mul_(scale).to(dt)
        s = {"case": dict(case), "x": normal(m, k), "w": normal(n, k, scale=k ** -0.5),
             "b": normal(n, scale=0.1) if case["bias"] else None, "res": normal(m, n) if case["res"] else None,
             "dy": normal(m, n) if case["train"] else None}
        s["leaves"] = [t for t in (s["x"], s["w"], s["b"], s["res"]) if t is not None]
        if case["train"]:
            for t in s["leaves"]:
                t.requires_grad_(True)
        return s
    if case["op"] in ("policy", "logprobs"):
        dt, b, t, v, pad = _DT[case["dtype"]], case["b"], case["t"], case["v"], case["pad"]
        actions = torch.randint(0, v - pad, (b, t), generator=g, device=dev)
        full = torch.empty(b, t + 1, v, dtype=dt, device=dev)   # a model's logits: one position more than targets
        for i in range(b):
            z = torch.randn(t + 1, v, generator=g, device=dev).mul_(2.0)
            if pad:
                z[:, v - pad:] = -math.inf                      # columns that fill the vocabulary up
            lift = torch.rand(t, 1, generator=g, device=dev).mul_(8.0).add_(2.0)
            z[:t].scatter_add_(1, actions[i].unsqueeze(1), lift)
            full[i] = z.to(dt)
        logits = full[:, :t]
        s = {"case": dict(case), "logits": logits, "actions": actions}
        if case["op"] == "logprobs":
            return s
        logp = torch.stack([z.float().log_softmax(-1).gather(1, a.unsqueeze(1)).squeeze(1)
                            for z, a in zip(logits, actions)])
        shift = torch.randn(b, t, generator=g, device=dev).mul_(0.15)
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):   # the clip's own borders say nothing
            shift = torch.where((shift - edge).abs() < 2e-3, shift + 5e-3, shift)
        s["old"] = logp - shift
        s["ref"] = logp + torch.randn(b, t, generator=g, device=dev).mul_(0.25)
        s["adv"] = torch.randn(b, t, generator=g, device=dev).add_(0.5)
        lengths = torch.randint(0 if b > 1 else 1, t + 1, (b,), generator=g, device=dev)
        lengths[b - 1] = t
        s["mask"] = torch.arange(t, device=dev).unsqueeze(0) < lengths.unsqueeze(1)
        s["logits"] = logits.requires_grad_(True)
        return s
    dt, gt, bits = _DT[case["dtype"]], _DT[_grad_type(case)], case["bits"]
    s = {"case": dict(case), "params": [], "grads": [], "state": [], "step": STEPS_DONE}
    for i, shape in enumerate(_shapes(case)):
        spread = torch.rand(shape[0], *([1] * (len(shape) - 1)), generator=g, device=dev).mul_(6).sub_(8).exp_()
        p = torch.randn(shape, generator=g, device=dev).mul_(0.02).to(dt)
        grad = (torch.randn(shape, generator=g, device=dev) * spread).to(gt)
        m = torch.randn(shape, generator=g, device=dev).mul_(0.3) * spread
        v = (torch.rand(shape, generator=g, device=dev).add_(0.5) * spread).square_()
        if bits == 8:
            m8, ms = _quantise_nearest(m)
            r8, rs = _quantise_nearest(v.sqrt_())
            st = {"exp_avg": m8, "exp_avg_scale": ms, "exp_rms": r8, "exp_rms_scale": rs}
        else:
            st = {"exp_avg": m, "exp_avg_sq": v}
        s["params"].append(p.requires_grad_(True))
        s["grads"].append(grad)
        s["state"].append(st)
    if own:   # the handle that a user's program keeps: the optimiser, continued from this state
        optim = _lvmhelpers("optim")
        opt = optim.AdamW(s["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits,
                          min_8bit_size=1, seed=SEED)
        for p, grad, st in zip(s["params"], s["grads"], s["state"]):
            opt.state[p].update(st, step=torch.full((), STEPS_DONE, dtype=torch.int64, device=dev))
            if gt == dt:
                p.grad = grad
        s["opt"], s["own_grads"] = opt, (None if gt == dt else s["grads"])   # (.grad has the weight's type)
    return s


def _quantise_nearest(x):
    """Starting values of an 8-bit state: (codes, scales), 256 values of the flattened tensor to a scale."""
    n = x.numel()
    y = torch.nn.functional.pad(x.reshape(-1), (0, -n % 256)).view(-1, 256)
    scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax(1, keepdim=True).clamp_min(1e-30) / 448.0)))
    codes = (y / scale).to(torch.float8_e4m3fn)
    return codes.view(-1)[:n].reshape(x.shape).contiguous(), scale.view(-1)


def _lvmhelpers(name):
    """A module of this repository's package (only ever called where `own` is true)."""
    import importlib
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-marginalization-lvm_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    return importlib.import_module("lvmhelpers." + name)


# --------------------------------------------------------------------------------------------- run
def run(s):
    op = s["case"]["op"]
    if own:
        return {"linear": _own_linear, "policy": _own_policy, "logprobs": _own_logprobs,
                "adamw": _own_adamw}[op](s)
    with torch.no_grad():
        return {"linear": _plain_linear, "policy": _plain_policy, "logprobs": _plain_logprobs,
                "adamw": _plain_adamw}[op](s)


def _own_linear(s):
    y = _lvmhelpers("functional").linear_act(s["x"], s["w"], s["b"], activation=s["case"]["act"], residual=s["res"])
    if not s["case"]["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, s["leaves"], s["dy"]))


def _act(name, h):
    if name == "none":
        return h
    if name == "relu":
        return torch.where(h > 0, h, torch.zeros_like(h))
    if name == "gelu":
        return 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
    if name == "tanh":
        return torch.tanh(h)
    sig = 1 / (1 + torch.exp(-h))
    return sig if name == "sigmoid" else h * sig


def _act_slope(name, h):
    if name == "none":
        return torch.ones_like(h)
    if name == "relu":
        return (h > 0).to(h.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    if name == "tanh":
        return 1 - torch.tanh(h) ** 2
    sig = 1 / (1 + torch.exp(-h))
    return sig * (1 - sig) if name == "sigmoid" else sig * (1 + h * (1 - sig))


def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    h = x @ w.t()
    if s["b"] is not None:
        h = h + s["b"].float()
    y = _act(case["act"], h)
    if s["res"] is not None:
        y = y + s["res"].float()
    y = y.to(dt)
    if not case["train"]:
        return [y]
    dh = s["dy"].float() * _act_slope(case["act"], h)
    out = [y, (dh @ w).to(dt), (dh.t() @ x).to(dt)]
    if s["b"] is not None:
        out.append(dh.sum(0).to(dt))
    if s["res"] is not None:
        out.append(s["dy"])
    return out


def _own_policy(s):
    loss, stats = _lvmhelpers("functional").clipped_policy_loss(
        s["logits"], s["actions"], s["old"], s["adv"], ref_logp=s["ref"], mask=s["mask"], clip_low=CLIP_LOW,
        clip_high=CLIP_HIGH, kl_coeff=KL, entropy_coeff=ENT, reduction=s["case"]["reduction"])
    (dlogits,) = torch.autograd.grad(loss, [s["logits"]])
    return {"loss": loss.detach(), "logp": stats["logp"], "entropy": stats["entropy"], "kl": stats["kl"],
            "clipped": stats["clipped"], "dlogits": dlogits}


def _own_logprobs(s):
    logp, entropy = _lvmhelpers("functional").token_logprobs(s["logits"], s["actions"])
    return {"logp": logp, "entropy": entropy}


def _plain_tokens(z, actions):
    """(softmax, log-softmax with 0 where the probability is 0, log-probability of the action, entropy)."""
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    p = e / total
    logs = torch.where(e > 0, z - top - torch.log(total), torch.zeros_like(z))
    logp = (z.gather(-1, actions.unsqueeze(-1)) - top).squeeze(-1).double() - torch.log(total.squeeze(-1).double())
    return p, logs, logp, -(p * logs).sum(-1)


def _plain_logprobs(s):
    _, _, logp, entropy = _plain_tokens(s["logits"].float(), s["actions"])
    return {"logp": logp.float(), "entropy": entropy}


def _plain_policy(s):
    z, mask = s["logits"].float(), s["mask"]
    p, logs, logp, entropy = _plain_tokens(z, s["actions"])
    adv = s["adv"].double()
    ratio = torch.exp(logp - s["old"].double())
    clipped = torch.where(adv > 0, ratio > 1 + CLIP_HIGH, (adv < 0) & (ratio < 1 - CLIP_LOW)) & mask
    surrogate = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    d = s["ref"].double() - logp
    kl = torch.exp(d) - d - 1
    per = torch.where(mask, surrogate + KL * kl - ENT * entropy.double(), torch.zeros_like(logp))
    norm = 1.0 / mask.sum().clamp_min(1).double() if s["case"]["reduction"] == "mean" else torch.ones((), dtype=torch.float64, device=z.device)
    loss = per.sum() * norm
    slope = torch.where(clipped, torch.zeros_like(ratio), -adv * ratio) + KL * (1 - torch.exp(d))
    zero = torch.zeros_like(entropy)
    c = torch.where(mask, (slope * norm).float(), zero).unsqueeze(-1)          # d loss / d logp
    h = torch.where(mask, (-ENT * norm).float().expand_as(entropy), zero).unsqueeze(-1)   # d loss / d entropy
    dz = -p * (c + h * (logs + entropy.unsqueeze(-1)))
    dz.scatter_add_(-1, s["actions"].unsqueeze(-1), c)
    keep = mask.to(torch.float32)
    return {"loss": loss.float(), "logp": torch.where(mask, logp.float(), zero), "entropy": entropy * keep,
            "kl": torch.where(mask, kl.float(), zero), "clipped": clipped, "dlogits": dz.to(s["logits"].dtype)}


def _own_adamw(s):
    s["opt"].step(grads=s["own_grads"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    """The optimiser's own buffers: weights and states, 8-bit states as their codes' values with the scales."""
    return [[p.detach() for p in s["params"]], [[st[k] for k in sorted(st) if k != "step"] for st in s["state"]]]


_C1, _C2, _M32 = 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _mix(x):
    """The rounding bits' hash, on whole numbers below 2^32 (Python's, or an int64 tensor's)."""
    x = x ^ (x >> 16)
    x = (x * _C1) & _M32
    x = x ^ (x >> 15)
    x = (x * _C2) & _M32
    return x ^ (x >> 16)


def _random_bits(n, index, step, dev):
    key = _mix((_mix((SEED + _C1 * step) & _M32) + index) & _M32)
    j = torch.arange(n, device=dev, dtype=torch.int64)
    return _mix(((j * _C1) & _M32).add_(key).bitwise_and_(_M32))


def _blocks(x, fill=0):
    return torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % 256), value=fill).view(-1, 256)


def _encode(x, bits, floor):
    """e4m3 codes and power-of-two scales of the 32-bit values x, rounded up with probability bits / 2^16;
    `floor`: values over zero keep at least the smallest code."""
    n, shape = x.numel(), x.shape
    x, bits = _blocks(x), _blocks(bits).double()
    _, k = torch.frexp(x.abs().amax(1, keepdim=True).double() / 448.0)
    scale = torch.exp2((k - (x.abs().amax(1, keepdim=True).double() <= 448.0 * torch.exp2(k.double() - 1)).to(k.dtype)).clamp_min(-100).double())
    y = x.abs().double() / scale
    _, e = torch.frexp(y)
    quantum = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    y = (torch.floor(y / quantum + bits / 65536.0) * quantum).clamp_max(448.0)
    if floor:
        y = torch.where(x > 0, y.clamp_min(2.0 ** -9), y)
    codes = torch.copysign(y, x.double()).float().to(torch.float8_e4m3fn)
    return codes.view(-1)[:n].reshape(shape), scale.float().view(-1)


def _decode(codes, scale):
    n = codes.numel()
    return (_blocks(codes.float()) * scale.view(-1, 1)).view(-1)[:n].reshape(codes.shape)


def _plain_adamw(s):
    s["step"] += 1
    t, (b1, b2) = s["step"], BETAS
    bc1, bc2 = 1 - b1 ** t, 1 - b2 ** t
    for i, (p, grad, st) in enumerate(zip(s["params"], s["grads"], s["state"])):
        if s["case"]["bits"] == 8:   # 64 bits, rounded once: the codes hang on these values
            g = grad.double()
            m = (_decode(st["exp_avg"], st["exp_avg_scale"]).double() * b1 + g * (1 - b1)).float()
            v = (_decode(st["exp_rms"], st["exp_rms_scale"]).double().square() * b2 + g.square() * (1 - b2)).float()
            bits = _random_bits(p.numel(), i, t, p.device)
            for key, x, u in (("exp_avg", m, bits & 0xFFFF), ("exp_rms", v.sqrt(), bits >> 16)):
                codes, scale = _encode(x, u, key == "exp_rms")
                st[key].copy_(codes)
                st[key + "_scale"].copy_(scale)
        else:
            g = grad.float()
            m = st["exp_avg"].mul_(b1).add_(g * (1 - b1))
            v = st["exp_avg_sq"].mul_(b2).add_(g * g * (1 - b2))
        w = p.float() * (1 - LR * DECAY)
        p.copy_(w - (LR / bc1) * m / (v.sqrt() / math.sqrt(bc2) + EPS))
    return _adamw_outputs(s)


# ------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _exact_linear, "policy": _exact_policy, "logprobs": _exact_policy,
                "adamw": _exact_adamw}[case["op"]](s)


def _exact_linear(s):
    case = s["case"]
    x, w = s["x"].double(), s["w"].double()
    h = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    if s["b"] is not None:
        h += s["b"].double()
    h += torch.mm(x, w.t().contiguous())
    name = case["act"]
    phi = 0.5 * torch.special.erfc(-h / math.sqrt(2.0))
    y = {"none": lambda: h, "relu": lambda: h.clamp_min(0), "gelu": lambda: h * phi, "tanh": lambda: torch.tanh(h),
         "sigmoid": lambda: torch.sigmoid(h), "silu": lambda: h * torch.sigmoid(h)}[name]()
    if s["res"] is not None:
        y = y + s["res"].double()
    if not case["train"]:
        return [y]
    sig = torch.sigmoid(h)
    slope = {"none": lambda: torch.ones_like(h), "relu": lambda: (h > 0).double(),
             "gelu": lambda: phi + h * torch.exp(-h.square() / 2) / math.sqrt(2 * math.pi),
             "tanh": lambda: 1 - torch.tanh(h).square(), "sigmoid": lambda: sig - sig.square(),
             "silu": lambda: sig + h * (sig - sig.square())}[name]()
    dh = s["dy"].double() * slope
    out = [y, torch.mm(dh, w), torch.mm(dh.t().contiguous(), x)]
    if s["b"] is not None:
        out.append(dh.sum(0))
    if s["res"] is not None:
        out.append(s["dy"].double())
    return out


def _exact_policy(s):
    case = s["case"]
    loss, count, rows = 0.0, 1, {"logp": [], "entropy": [], "kl": []}
    train = case["op"] == "policy"
    if train and case["reduction"] == "mean":
        count = max(1, int(s["mask"].sum()))
    whole = s["logits"].numel() * 8 <= 16 << 30
    dz = torch.empty(s["logits"].shape, dtype=torch.float64 if whole else torch.float32, device="cuda") if train else None
    for i in range(case["b"]):
        lsm = torch.log_softmax(s["logits"][i].detach().double(), -1)
        p = lsm.exp()
        plogp = torch.special.entr(p)
        ent = plogp.sum(-1)
        at = s["actions"][i].unsqueeze(-1)
        logp = lsm.gather(-1, at).squeeze(-1)
        if not train:
            rows["logp"].append(logp)
            rows["entropy"].append(ent)
            continue
        live = s["mask"][i].double()
        adv, old, ref = (s[k][i].double() for k in ("adv", "old", "ref"))
        ratio = (logp - old).exp()
        free = torch.where(adv >= 0, ratio <= 1 + CLIP_HIGH, ratio >= 1 - CLIP_LOW).double()
        bounded = torch.where(adv >= 0, ratio.clamp_max(1 + CLIP_HIGH), ratio.clamp_min(1 - CLIP_LOW))
        kl = torch.expm1(ref - logp) - (ref - logp)
        loss += float(((-adv * bounded + KL * kl - ENT * ent) * live).sum()) / count
        c = (-adv * ratio * free - KL * torch.expm1(ref - logp)) * live / count
        h = -ENT * live / count
        d = -c.unsqueeze(-1) * p + h.unsqueeze(-1) * (plogp - p * ent.unsqueeze(-1))
        dz[i] = d.scatter_add_(-1, at, c.unsqueeze(-1))
        rows["logp"].append(logp * live)
        rows["entropy"].append(ent * live)
        rows["kl"].append(kl * live)
    out = {k: torch.stack(v) for k, v in rows.items() if v}
    if train:
        out.update(loss=torch.tensor(loss, dtype=torch.float64), dlogits=dz, clipped=None)
    return out


def _between_codes(x, bits):
    """The same rounding from the other side: of the two neighbours in the list of all e4m3 values, the
    upper one if the distance to the lower, in units of the gap, and bits / 2^16 reach 1 together."""
    table = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    top = _blocks(x.abs()).amax(1, keepdim=True)
    powers = torch.exp2(torch.arange(-100, 121, dtype=torch.float64, device=x.device))
    scale = powers[torch.searchsorted(powers * 448.0, top).clamp_max(220)]
    y = (_blocks(x.abs()) / scale).view(-1)[:x.numel()]
    low = (torch.searchsorted(table, y, right=True) - 1).clamp_max(125)
    gap = table[low + 1] - table[low]
    up = (y - table[low]) / gap + bits.reshape(-1) / 65536.0 >= 1
    value = torch.where(y >= 448.0, 448.0, table[low + up.long()]).reshape(x.shape)
    return torch.where(x < 0, -value, value), scale.view(-1)


def _exact_adamw(s):
    t, (b1, b2) = s["step"] + 1, BETAS
    weights, states = [], []
    for i, (p, grad, st) in enumerate(zip(s["params"], s["grads"], s["state"])):
        g = grad.double()
        if s["case"]["bits"] == 8:
            # by definition the averages of an 8-bit state are rounded to 32 bits before they are encoded
            m = torch.lerp(g, _decode(st["exp_avg"], st["exp_avg_scale"]).double(), b1).float().double()
            v = torch.lerp(g ** 2, _decode(st["exp_rms"], st["exp_rms_scale"]).double() ** 2, b2).float().double()
            bits = _random_bits(p.numel(), i, t, p.device)
            m8, ms = _between_codes(m, bits % 65536)
            r8, rs = _between_codes(v.sqrt().float().double(), bits // 65536)
            r8 = torch.where((v > 0) & (r8 == 0), 2.0 ** -9, r8)
            states.append([m8, ms, r8, rs])
        else:
            m = torch.lerp(g, st["exp_avg"].double(), b1)
            v = torch.lerp(g ** 2, st["exp_avg_sq"].double(), b2)
            states.append([m, v])
        unbiased = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
        weights.append(p.double() - LR * DECAY * p.double() - LR * unbiased)
    return [weights, states]
