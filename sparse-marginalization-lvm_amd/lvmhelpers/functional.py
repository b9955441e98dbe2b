"""torch.autograd glue over the C-ABI kernels (``_native``).  Host-side plumbing only."""
import torch

from . import _native


def _patterns_written(x, p, mask):
    """Did this forward call leave every row's 16-bit-per-lane pattern in `mask`?  Only the vector
    path of the 16-register tiles does (32 < K <= 1024, K % 4 == 0, x and p 16-byte aligned); the
    pattern-fed compaction must not be handed a buffer that was never filled."""
    K = x.shape[-1]
    return (mask is not None and 32 < K <= 1024 and K % 4 == 0
            and x.data_ptr() % 16 == 0 and p.data_ptr() % 16 == 0)


class _Sparsemax(torch.autograd.Function):
    """Row-wise sparsemax over the last dim (replaces entmax.sparsemax; marg.py:45,51)."""

    @staticmethod
    def forward(ctx, x):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1])
        p, supp, _, _, _, cols, mask = _native.sparsemax_fwd(x2, want_cols=True, want_mask=True)
        ctx.has_mask = mask is not None
        ctx.save_for_backward(p, supp, cols, *([mask] if mask is not None else []))
        ctx.mark_non_differentiable(cols)
        patterns = mask if _patterns_written(x2, p, mask) else None
        if patterns is not None:
            ctx.mark_non_differentiable(patterns)
        return p.view(shape), cols, patterns

    @staticmethod
    def backward(ctx, dy, _dcols=None, _dpatterns=None):
        p, supp, cols = ctx.saved_tensors[:3]
        mask = ctx.saved_tensors[3] if ctx.has_mask else None
        dx = _native.sparsemax_bwd_cols(dy.reshape(p.shape).contiguous(), cols, p, supp, mask)
        return dx.view(dy.shape)


class _Entmax15(torch.autograd.Function):
    """Row-wise 1.5-entmax over the last dim (replaces entmax.entmax15; marg.py:46)."""

    @staticmethod
    def forward(ctx, x):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1])
        ctx.listed = _native.entmax15_has_lists(shape[-1]) and x2.shape[0] > 0
        if ctx.listed:   # rows of one wave: the forward leaves each row's support list and sqrt(p)
            p, cols, vals = _native.entmax15_fwd_lists(x2)
            ctx.save_for_backward(p, cols, vals)
        else:
            p, _, _ = _native.entmax15_fwd(x2)
            ctx.save_for_backward(p)
        return p.view(shape)

    @staticmethod
    def backward(ctx, dy):
        p = ctx.saved_tensors[0]
        dy2 = dy.reshape(p.shape).contiguous()
        if ctx.listed:
            return _native.entmax15_bwd_lists(dy2, p, ctx.saved_tensors[1], ctx.saved_tensors[2]).view(dy.shape)
        return _native.entmax15_bwd(dy2, p).view(dy.shape)


class _SparsemaxEntropy(torch.autograd.Function):
    """Fused sparsemax + Shannon entropy (marg.py:51-52): one forward kernel, one backward kernel."""

    @staticmethod
    def forward(ctx, x):
        p, supp, _, _, ent, cols, mask = _native.sparsemax_fwd(x, want_entropy=True, want_cols=True,
                                                               want_mask=True)
        ctx.has_mask = mask is not None
        ctx.save_for_backward(p, supp, cols, *([mask] if mask is not None else []))
        ctx.mark_non_differentiable(supp, cols)
        patterns = mask if _patterns_written(x, p, mask) else None
        if patterns is not None:
            ctx.mark_non_differentiable(patterns)
        return p, ent, supp, cols, patterns

    @staticmethod
    def backward(ctx, dp, dent, _dsupp, _dcols=None, _dpatterns=None):
        p, supp, cols = ctx.saved_tensors[:3]
        mask = ctx.saved_tensors[3] if ctx.has_mask else None
        if dp is None and dent is None:
            return torch.zeros_like(p)
        if dent is None:
            g = dp
        elif dp is None:
            g = _entropy_vjp(p, dent)
        else:
            g = dp + _entropy_vjp(p, dent)
        return _native.sparsemax_bwd_cols(g.contiguous(), cols, p, supp, mask)


def _entropy_vjp(p, dent):
    # d/dp of -sum_{p>0} pc*log(pc), pc = clamp(p, eps, 1-eps): the clamp passes gradient only
    # inside [eps, 1-eps] (marg.py:18-28)
    eps = torch.finfo(p.dtype).eps
    inside = (p >= eps) & (p <= 1 - eps)
    safe = torch.where(inside, p, torch.ones_like(p))
    return torch.where(inside, -(safe.log() + 1.0), torch.zeros_like(p)) * dent.unsqueeze(-1)


class _Entropy(torch.autograd.Function):
    """lvmhelpers/marg.py:6-28 on an arbitrary probability matrix."""

    @staticmethod
    def forward(ctx, p):
        ctx.save_for_backward(p)
        return _native.entropy(p)

    @staticmethod
    def backward(ctx, dent):
        (p,) = ctx.saved_tensors
        return _entropy_vjp(p, dent)


class _WeightedLossReduce(torch.autograd.Function):
    """inv_b * <vals, comps> with the fused deterministic reduction kernel (marg.py:125-126,
    structmarg.py:140,242)."""

    @staticmethod
    def forward(ctx, vals, comps, inv_b):
        total, _ = _native.weighted_loss_reduce_fwd(vals, comps, None, inv_b)
        ctx.save_for_backward(vals, comps)
        ctx.inv_b = inv_b
        return total.reshape(())

    @staticmethod
    def backward(ctx, g):
        vals, comps = ctx.saved_tensors
        dv, dc = _native.weighted_loss_reduce_bwd(
            vals, comps, g.to(torch.float32), ctx.inv_b,
            want_dvals=ctx.needs_input_grad[0], want_dcomps=ctx.needs_input_grad[1])
        return dv, dc, None


class _SupportEntropy(torch.autograd.Function):
    """-inv_b * sum_{p > 0} p log p in two launches forward and one backward (structmarg.py:51-54,
    200: seven elementwise launches forward, six backward, at batch 64 all of them launch latency)."""

    @staticmethod
    def forward(ctx, p, inv_b):
        p = p.contiguous()
        ctx.save_for_backward(p)
        ctx.inv_b = inv_b
        return _native.support_entropy_fwd(p, inv_b).reshape(())

    @staticmethod
    def backward(ctx, g):
        (p,) = ctx.saved_tensors
        return _native.support_entropy_bwd(p, g.to(torch.float32), ctx.inv_b), None


def support_entropy(p, inv_b=1.0):
    """-(p[p > 0] @ log p[p > 0]) * inv_b as a 0-d tensor (no clamping: structmarg.py:51-54, 200)."""
    return _SupportEntropy.apply(p, float(inv_b))


class _GatherSupport(torch.autograd.Function):
    """vals = p[rows, cols] for the compaction's (rows, cols), whose values the compaction kernel has
    already written: the forward launches nothing, the backward is one scatter of distinct
    positions (torch's index backward zero-fills, sorts the indices and accumulates: 7 launches)."""

    @staticmethod
    def forward(ctx, p, row_offsets, cols, vals):
        ctx.save_for_backward(row_offsets, cols)
        ctx.shape = tuple(p.shape)
        return vals.view_as(vals)

    @staticmethod
    def backward(ctx, g):
        row_offsets, cols = ctx.saved_tensors
        R, K = ctx.shape
        return _native.support_scatter(g.contiguous(), row_offsets, cols, R, K), None, None, None


class _GatherRows(torch.autograd.Function):
    """table[rows] for the compaction's (sorted, row-major) rows.  The backward sums each row's
    entries in order with one kernel (smlvm_support_segment_sum) instead of torch's index_select
    backward, which adds with float atomics in an order that changes from run to run."""

    @staticmethod
    def forward(ctx, table, rows, row_offsets):
        ctx.save_for_backward(row_offsets)
        ctx.R = table.shape[0]
        return table.index_select(0, rows)

    @staticmethod
    def backward(ctx, g):
        (row_offsets,) = ctx.saved_tensors
        return _native.support_segment_sum(g.contiguous(), row_offsets, ctx.R), None, None


def gather_rows(table, rows, row_offsets):
    """table [R, ...] gathered at the compaction's rows [N] (int64, row-major order) with a
    deterministic backward; row_offsets [R+1] are the compaction's."""
    return _GatherRows.apply(table, rows, row_offsets)


def gather_support(p, row_offsets, cols, vals):
    """The compacted probabilities `vals` (== p[rows, cols], row-major) as a differentiable function
    of p [R, K]."""
    return _GatherSupport.apply(p, row_offsets, cols, vals)


class _SparseMAP(torch.autograd.Function):
    """Batched bit-vector SparseMAP (sparsemap.py:12-44 for every sample of the batch at once)."""

    @staticmethod
    def forward(ctx, scores, init_scores, budget, max_iter):
        out = _native.sparsemap_fwd(scores.detach(), init_scores, budget, max_iter)
        ctx.n = scores.shape[1]
        ctx.save_for_backward(out["aset_bits"], out["alen"], out["inv_a"])
        for k in ("aset_bits", "alen", "iters", "status"):
            ctx.mark_non_differentiable(out[k])
        return out["p"], out["aset_bits"], out["alen"], out["iters"], out["status"]

    @staticmethod
    def backward(ctx, dp, *_):
        aset_bits, alen, inv_a = ctx.saved_tensors
        return _native.sparsemap_bwd(dp.contiguous(), aset_bits, alen, inv_a, ctx.n), None, None, None


class _LowRankCE(torch.autograd.Function):
    """sum_f cross_entropy(x[n,f,:] @ w.T + b, y[n,f]) without the [N,F,C] logits
    (experiments/bit_vector-vae/archs.py:26-29 + train.py:361-371)."""

    @staticmethod
    def forward(ctx, x, w, b, y):
        # when x wants a gradient the forward pass also leaves d loss / d x (R packed FMAs more per
        # logit): the backward's dX is then an elementwise product, not a third pass of exponentials
        ctx.has_dxdir = bool(ctx.needs_input_grad[0]) and x.numel() > 0
        if ctx.has_dxdir:
            loss, lse, _, dxdir = _native.lowrank_ce_fwd(x, w, b, y, want_dxdir=True)
            ctx.save_for_backward(x, w, b, y, lse, dxdir)
        else:
            loss, lse, _ = _native.lowrank_ce_fwd(x, w, b, y)
            ctx.save_for_backward(x, w, b, y, lse)
        return loss

    @staticmethod
    def backward(ctx, gloss):
        x, w, b, y, lse = ctx.saved_tensors[:5]
        gloss = gloss.contiguous().to(torch.float32)
        want_dw = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        if ctx.has_dxdir:
            dx = ctx.saved_tensors[5] * gloss.view(-1, 1, 1) if ctx.needs_input_grad[0] else None
            dw = db = None
            if want_dw:
                _, dw, db = _native.lowrank_ce_bwd(x, w, b, y, lse, gloss, want_dx=False, want_dw=True)
            return dx, dw, db, None
        dx, dw, db = _native.lowrank_ce_bwd(x, w, b, y, lse, gloss,
                                            want_dx=ctx.needs_input_grad[0], want_dw=want_dw)
        return dx, dw, db, None


def lowrank_categorical_nll(x, w, b, y):
    """x [N,F,R], w [C,R], b [C], y [N,F] integer labels -> per-row loss [N]."""
    return _LowRankCE.apply(x.contiguous(), w.contiguous(), b.contiguous(), y)


def linear_act(x, weight, bias=None, activation="none", residual=None):
    """activation(x @ weight.T + bias) + residual as one kernel (split over the inner axis: two).

    x [..., K], weight [N, K], bias [N], residual [..., N]: float32, float16 or bfloat16, all of one type, on one
    GPU; residual has exactly the output's shape (nothing is broadcast).  activation: 'none', 'relu', 'gelu' (the erf
    form), 'silu', 'sigmoid', 'tanh'.  Products are summed in fp32; float32 operands are multiplied to
    fp32 accuracy on the bf16 matrix cores (an infinite operand may then give NaN instead of an
    infinity).  Differentiable in all four, once and in reverse mode; `bias`' gradient comes from the pass that
    applies the activation's slope, without an activation from the one that computes `weight`'s."""
    name = "linear_act"
    act = _native.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{name}: activation must be one of {sorted(_native.ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{name}: x [..., K] and weight [N, K] do not fit: {tuple(x.shape)}, {tuple(weight.shape)}")
    out_shape = x.shape[:-1] + weight.shape[:1]
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"{name}: bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != out_shape:
        raise ValueError(f"{name}: residual must be {tuple(out_shape)}, got {tuple(residual.shape)}")
    if not x.is_cuda:
        raise _native.NativeError(f"{name}: expected GPU tensors (the hot path has no CPU fallback)")
    dtype, at = x.dtype, x.get_device()
    if dtype not in _native.KINDS:
        raise TypeError(f"{name}: expected float32, float16 or bfloat16, got {dtype}")
    for t, what in ((weight, "weight"), (bias, "bias"), (residual, "residual")):
        if t is not None and (t.dtype != dtype or t.get_device() != at):       # (-1 on the CPU)
            raise TypeError(f"{name}: {what} must have x's type and device ({x.dtype}, {x.device}), got {t.dtype}, {t.device}")
    if x.dim() != 2:
        x = x.reshape(-1, weight.shape[1]) if x.numel() else x.reshape(out_shape[:-1].numel(), weight.shape[1])
    if residual is not None and residual.dim() != 2:
        residual = residual.reshape(x.shape[0], weight.shape[0])
    if bias is not None:
        bias = bias.contiguous()
    y = _native.autograd().linear_act(x, weight, bias, residual, act)
    return y if len(out_shape) == 2 else y.view(out_shape)


def _policy_rows(logits, actions, name):
    """logits [..., V] -> [B, T, V] without a copy where the strides allow it, actions -> [B, T] int64."""
    if logits.dim() < 2 or logits.shape[-1] < 1:
        raise ValueError(f"{name}: logits must be [..., V] with at least one leading axis and V >= 1")
    lead = logits.shape[:-1]
    if actions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name}: actions must be int64 or int32, got {actions.dtype}")
    if logits.dim() == 2:
        logits = logits.unsqueeze(0)
    elif logits.dim() > 3:
        logits = logits.reshape(-1, logits.shape[-2], logits.shape[-1])
    return logits, _row_values(actions, lead, logits, name, "actions", torch.int64)


def _row_values(t, lead, logits, name, what, dtype):
    if t.shape != lead:
        raise ValueError(f"{name}: {what} must have logits' leading shape {tuple(lead)}, got {tuple(t.shape)}")
    if t.device != logits.device:
        raise _native.NativeError(f"{name}: {what} must be on the logits' device")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: {what} is a constant of the loss; detach it (no gradient would reach it)")
    if t.dtype != dtype:
        if dtype == torch.float32 and t.dtype not in _NARROW:
            raise TypeError(f"{name}: {what} must be float32, float16 or bfloat16, got {t.dtype}")
        t = t.to(dtype)
    if t.requires_grad:          # (gradients are off)
        t = t.detach()
    shape = logits.shape[:2]
    return (t if t.shape == shape else t.reshape(shape)).contiguous()


def _row_mask(mask, lead, logits, name):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"{name}: mask must be bool or uint8, got {mask.dtype}")
    return _row_values(mask, lead, logits, name, "mask", mask.dtype).view(torch.uint8)


def token_logprobs(logits, actions, mask=None):
    """logits [..., V] (float32, float16, bfloat16), actions [...] integers -> (logp [...], entropy [...]) in
    float32: the log-probability of each action under softmax(logits) and each row's entropy, without
    a [..., V] intermediate; differentiable in logits.

    -inf logits have probability zero; a row without a finite logit, with a NaN or +inf one, or with an
    action outside [0, V) gives NaN.  mask (bool or uint8 [...]): rows that are False are not read and
    give 0.  Leading axes may be strided (a shifted slice of a model's output is not copied)."""
    rows, act = _policy_rows(logits, actions, "token_logprobs")
    lead = logits.shape[:-1]
    mask = _row_mask(mask, lead, rows, "token_logprobs")
    _native.need_logits(rows)
    logp, entropy = _native.autograd().token_logprobs(rows, act, mask)
    return logp.view(lead), entropy.view(lead)


def clipped_policy_loss(logits, actions, old_logp, advantages, ref_logp=None, mask=None, clip_low=0.2, clip_high=0.2,
                        kl_coeff=0.0, entropy_coeff=0.0, reduction="mean"):
    """Clipped policy-gradient loss of a discrete policy, with a KL term to a reference policy and an
    entropy bonus, straight from the logits:

        ratio = exp(logp - old_logp),   d = ref_logp - logp
        l = -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coeff (e^d - d - 1) - entropy_coeff H

    averaged over (reduction="mean") or summed over (="sum") the rows with mask True.

    logits [..., V]; actions, old_logp, advantages, ref_logp, mask [...].  Only logits get a gradient;
    the others are constants (one that requires a gradient is refused).  Returns (loss, stats) with
    stats = {'logp', 'entropy', 'kl' (float32), 'clipped' (bool)}, all [...] and without gradient; masked
    rows are not read, hold zeros there and get a zero gradient.  Other conventions as in `token_logprobs`.

    When logits require a gradient, it is computed in the forward pass (one read of the logits and
    one write, instead of two reads and one write): memory for it is taken there."""
    name = "clipped_policy_loss"
    if reduction not in ("mean", "sum"):
        raise ValueError(f"{name}: reduction must be 'mean' or 'sum', got {reduction!r}")
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError(f"{name}: need 0 <= clip_low <= 1 and clip_high >= 0, got {clip_low}, {clip_high}")
    if ref_logp is None and kl_coeff != 0.0:
        raise ValueError(f"{name}: kl_coeff needs ref_logp")
    rows, act = _policy_rows(logits, actions, name)
    lead = logits.shape[:-1]
    f32 = torch.float32
    old = _row_values(old_logp, lead, rows, name, "old_logp", f32)
    adv = _row_values(advantages, lead, rows, name, "advantages", f32)
    ref = None if ref_logp is None else _row_values(ref_logp, lead, rows, name, "ref_logp", f32)
    mask = _row_mask(mask, lead, rows, name)
    _native.need_logits(rows)
    loss, logp, entropy, kl, clipped = _native.autograd().clipped_policy_loss(
        rows, act, old, adv, ref, mask, float(clip_low), float(clip_high),
        float(kl_coeff), float(entropy_coeff), reduction == "mean")
    stats = {"logp": logp, "entropy": entropy, "kl": kl, "clipped": clipped}
    return loss, stats if len(lead) == 2 else {k: v.view(lead) for k, v in stats.items()}


_NARROW = (torch.float16, torch.bfloat16)


def sparsemax(X, dim=-1):
    """entmax.sparsemax replacement: Euclidean projection of each slice along `dim` onto the simplex.
    The kernels compute in fp32; half / bfloat16 inputs (autocast) are widened, and the result
    comes back in the input's dtype (float64 is refused rather than silently narrowed)."""
    if X.dtype in _NARROW:
        return sparsemax(X.float(), dim).to(X.dtype)
    if dim < 0:
        dim += X.dim()
    if dim != X.dim() - 1:
        return _Sparsemax.apply(X.transpose(dim, -1).contiguous())[0].transpose(dim, -1)
    p, cols, patterns = _Sparsemax.apply(X.contiguous())
    if p.dim() == 2:
        _tag_support(p, cols, patterns)
    return p


def entmax15(X, dim=-1):
    """entmax.entmax15 replacement: p = max(X/2 - tau, 0)^2 along `dim`, sum p = 1 (fp32 kernels;
    half / bfloat16 inputs are widened as in `sparsemax`)."""
    if X.dtype in _NARROW:
        return entmax15(X.float(), dim).to(X.dtype)
    if dim < 0:
        dim += X.dim()
    if dim != X.dim() - 1:
        return _Entmax15.apply(X.transpose(dim, -1).contiguous()).transpose(dim, -1)
    return _Entmax15.apply(X.contiguous())


SUPPORT_ATTR = "_smlvm_support_cols"


def _tag_support(p, cols, patterns=None):
    """Hang the forward's support lists on the probability tensor itself, so that a later
    `_native.support_compact(p.detach(), support_cols=support_cols_of(p))` does not have to scan p
    again.  The tag lives on this tensor object only (views, detach() and arithmetic drop it) and
    records the tensor's storage and version counter: an in-place change of p afterwards (masking,
    renormalising, clamp_) makes the lists stale, and support_cols_of then returns None.
    patterns: the forward's 16-bit-per-lane non-zero patterns, when it wrote them (rows without a
    list are then counted from those instead of from p: `support_mask_of`)."""
    setattr(p, SUPPORT_ATTR, (cols, p.data_ptr(), p._version, patterns))


def _support_tag(p):
    tag = getattr(p, SUPPORT_ATTR, None)
    if tag is None:
        return None
    cols, ptr, version, patterns = tag
    if p.dim() != 2 or cols.shape[0] != p.shape[0] or p.data_ptr() != ptr or p._version != version:
        return None
    return cols, patterns


def support_cols_of(p):
    tag = _support_tag(p)
    return None if tag is None else tag[0]


def support_mask_of(p):
    """The forward's patterns for `_native.support_compact(..., support_mask=...)`, or None."""
    tag = _support_tag(p)
    return None if tag is None else tag[1]


def sparsemax_with_entropy(X):
    """X [B,K] -> (p [B,K], entropy [B], supp_size [B] int32)."""
    p, ent, supp, cols, patterns = _SparsemaxEntropy.apply(X.contiguous())
    _tag_support(p, cols, patterns)
    return p, ent, supp


def entropy(p):
    return _Entropy.apply(p.contiguous())


def weighted_loss(vals, comps, inv_b):
    """inv_b * sum_j vals[j]*comps[j] as a 0-d tensor (differentiable in both)."""
    return _WeightedLossReduce.apply(vals.contiguous(), comps.contiguous(), float(inv_b))


def sparsemap_batched(scores, init_scores=None, budget=0, max_iter=300):
    """scores [B,n] -> (p [B,n+1] differentiable, aset_bits, alen, iters, status)."""
    return _SparseMAP.apply(scores.contiguous(), init_scores, int(budget), int(max_iter))
