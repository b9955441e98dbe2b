"""CPU: what token_logprobs / clipped_policy_loss and their C entries refuse, before a GPU is touched."""
import ctypes

import pytest
import torch

from lvmhelpers import _native
from lvmhelpers import functional as F_


def _args(**over):
    d = dict(logits=torch.zeros(2, 3, 5), actions=torch.zeros(2, 3, dtype=torch.int64), old_logp=torch.zeros(2, 3),
             advantages=torch.zeros(2, 3))
    d.update(over)
    return d


@pytest.mark.parametrize("over,error", [
    (dict(), _native.NativeError),                                             # CPU tensors
    (dict(logits=torch.zeros(5)), ValueError),
    (dict(logits=torch.zeros(2, 3, 0)), ValueError),
    (dict(actions=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(actions=torch.zeros(2, 3)), TypeError),
    (dict(old_logp=torch.zeros(2)), ValueError),
    (dict(advantages=torch.zeros(2, 3, requires_grad=True)), ValueError),
    (dict(ref_logp=torch.zeros(3, 2)), ValueError),
    (dict(old_logp=torch.zeros(2, 3, dtype=torch.float64)), TypeError),
    (dict(advantages=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
    (dict(mask=torch.zeros(2, 3)), TypeError),
    (dict(mask=torch.zeros(2, dtype=torch.bool)), ValueError),
    (dict(kl_coeff=0.1), ValueError),
    (dict(clip_low=-0.1), ValueError), (dict(clip_low=1.5), ValueError), (dict(clip_high=float("nan")), ValueError),
    (dict(reduction="none"), ValueError),
])
def test_policy_loss_refuses(over, error):
    with pytest.raises(error):
        F_.clipped_policy_loss(**_args(**over))


def test_logprobs_refuse():
    with pytest.raises(_native.NativeError):
        F_.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        F_.token_logprobs(torch.zeros(2, 5), torch.zeros(3, dtype=torch.int64))


def test_c_entries_check_their_arguments():
    L = _native.lib()
    i64, i32, f32, sz = ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_size_t
    one = ctypes.c_void_p(16)

    def fwd(z=one, kind=0, a=one, B=2, T=3, V=5):
        return L.smlvm_token_logprobs_fwd(z, i32(kind), i64(15), i64(5), a, None, one, one, one, i64(B), i64(T), i64(V), None)
    assert fwd(B=0) == 0 and fwd(T=0) == 0
    assert fwd(z=None) == -1 and fwd(a=None) == -1 and fwd(V=0) == -1 and fwd(kind=3) == -1 and fwd(B=-1) == -1
    assert fwd(B=1 << 20, T=1 << 20) == -2 and fwd(V=1 << 31) == -2

    def bwd(stats=one, c=one, g=one, keep=0, out=one, B=2):
        return L.smlvm_token_logprobs_bwd(one, i32(0), i64(15), i64(5), one, None, stats, c, None, g, i32(keep), out, i64(B),
                                          i64(3), i64(5), None)
    assert bwd(B=0) == 0
    assert bwd(stats=None) == -1 and bwd(c=None) == -1 and bwd(out=None) == -1 and bwd(g=None, keep=1) == -1
    need = L.smlvm_policy_loss_workspace_bytes(6)

    def loss(low=0.2, high=0.2, out=one, old=one, ws=one, nbytes=need, B=2, c=one):
        return L.smlvm_policy_loss(one, i32(0), i64(15), i64(5), one, None, old, one, None, f32(low), f32(high), f32(0), f32(0),
                                   i32(1), out, one, one, None, None, one, c, one, None, i64(B), i64(3), i64(5), ws,
                                   sz(nbytes), None)
    assert loss(low=-0.1) == -1 and loss(high=float("nan")) == -1 and loss(out=None) == -1 and loss(old=None) == -1
    assert loss(c=None) == -1 and loss(B=-1) == -1
    assert loss(ws=None) == -4 and loss(nbytes=need - 1) == -4
    assert L.smlvm_stream_capture_id(None, None) == -1
