"""CPU: what linear_act, its module and its C entries refuse."""
import ctypes

import pytest
import torch

from lvmhelpers import _native, fused
from lvmhelpers import functional as F_


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(2, 3), torch.zeros(4, 3)), _native.NativeError),
    ((torch.zeros(2, 3), torch.zeros(4, 5)), ValueError),
    ((torch.zeros(2, 3), torch.zeros(3)), ValueError),
    ((torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(3)), ValueError),
    ((torch.zeros(2, 3), torch.zeros(4, 3), None, "softplus"), ValueError),
    ((torch.zeros(2, 3), torch.zeros(4, 3), None, "none", torch.zeros(4)), ValueError),       # no broadcasting
    ((torch.zeros(2, 3), torch.zeros(4, 3), None, "none", torch.zeros(1, 4)), ValueError),
])
def test_refusals(args, error):
    with pytest.raises(error):
        F_.linear_act(*args)


def test_module_refuses_unknown_activations():
    with pytest.raises(ValueError):
        fused.LinearAct(3, 4, activation="softplus")
    assert list(fused.LinearAct(3, 4, activation="relu").state_dict()) == ["weight", "bias"]


def test_fuse_linears_leaves_hooks_and_subclasses():
    class Mine(torch.nn.Linear):
        pass
    hooked = torch.nn.Linear(3, 3)
    hooked.register_forward_hook(lambda *a: None)
    act = torch.nn.ReLU()
    act.register_forward_hook(lambda *a: None)
    net = fused.fuse_linears(torch.nn.Sequential(Mine(3, 3), hooked, torch.nn.Linear(3, 3), act, torch.nn.Linear(3, 2)))
    assert type(net[0]) is Mine and net[1] is hooked and net[2].activation == "none" and net[3] is act
    assert type(net[4]) is fused.LinearAct

    class Branches(torch.nn.Sequential):
        def forward(self, x):
            return sum(m(x) for m in self)
    assert type(fused.fuse_linears(Branches(torch.nn.Linear(3, 3), torch.nn.ReLU()))[0]) is torch.nn.Linear
    assert type(fused.fuse_linears(torch.nn.Sequential(torch.nn.Linear(3, 3).double()))[0]) is torch.nn.Linear
    back = torch.nn.Linear(3, 3)
    back.register_full_backward_hook(lambda *a: None)
    assert fused.fuse_linears(torch.nn.Sequential(back))[0] is back


def test_c_entries_check_their_arguments():
    L = _native.lib()
    i64, i32, sz = ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t
    one = ctypes.c_void_p(16)
    big = L.smlvm_linear_fwd_workspace_bytes(0, 5, 64, 100000)
    assert big > 0 and L.smlvm_linear_bwd_workspace_bytes(0, 2, 4, 4, 4) >= 64               # (dh)
    assert L.smlvm_linear_fwd_workspace_bytes(7, 4, 4, 4) == 0 and L.smlvm_linear_bwd_workspace_bytes(7, 0, 4, 4, 4) == 0
    for sizes in ((0, 4, 4), (4, 0, 4), (4, 4, 0), (0, 0, 0)):                                # empty axes
        assert L.smlvm_linear_fwd_workspace_bytes(0, *sizes) >= 0 and L.smlvm_linear_bwd_workspace_bytes(2, 1, *sizes) >= 0

    def fwd(x=one, ldx=100000, w=one, y=one, kind=0, act=0, M=5, N=64, K=100000, ws=one, nbytes=big, r=None, ldr=64):
        return L.smlvm_linear_fwd(x, i64(ldx), w, i64(max(K, 1)), None, r, i64(ldr), y, None, i32(kind), i32(act), i64(M), i64(N),
                                  i64(K), ws, sz(nbytes), None)
    assert fwd(M=0) == 0 and fwd(N=0) == 0
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(y=None) == -1 and fwd(kind=3) == -1 and fwd(act=6) == -1
    assert fwd(ldx=99999) == -1 and fwd(r=one, ldr=63) == -1 and fwd(M=-1) == -1 and fwd(M=1 << 31) == -2
    assert fwd(ws=None, nbytes=0) == -4 and fwd(nbytes=1) == -4                    # the split product's partial sums

    need = L.smlvm_linear_bwd_workspace_bytes(0, 1, 4, 4, 4)

    def bwd(dy=one, ldy=4, h=one, h_is_y=0, x=one, w=one, dx=one, dw=one, db=one, act=1, M=4, ws=one, nbytes=need):
        return L.smlvm_linear_bwd(dy, i64(ldy), h, i32(h_is_y), x, i64(4), w, i64(4), dx, dw, db, i32(0), i32(act), i64(M), i64(4),
                                  i64(4), ws, sz(nbytes), None)
    assert bwd(M=-1) == -1 and bwd(act=7) == -1 and bwd(dy=None) == -1 and bwd(h=None) == -1 and bwd(x=None) == -1
    assert bwd(w=None) == -1 and bwd(dw=None) == -1 and bwd(ldy=5) == -1 and bwd(ldy=3) == -1
    assert bwd(act=2, h_is_y=1) == -1                                                          # y stands in for relu only
    assert bwd(ws=None) == -4 and bwd(nbytes=8) == -4
    assert bwd(dx=None, dw=None, db=None, act=0) == 0                                          # nothing wanted


def test_launches_of_too_many_threads_are_refused():
    L = _native.lib()
    i64, i32 = ctypes.c_int64, ctypes.c_int32
    one, most = ctypes.c_void_p(16), (1 << 31) - 1
    for kind in (0, 1, 2):
        for M, N in ((1, most), (4, most), (most, 1)):
            assert L.smlvm_linear_fwd_workspace_bytes(kind, M, N, 1) == 0
            assert L.smlvm_linear_fwd(one, i64(1), one, i64(1), None, None, i64(N), one, None, i32(kind), i32(0), i64(M), i64(N),
                                      i64(1), None, ctypes.c_size_t(0), None) == -2
        assert L.smlvm_linear_bwd(one, i64(1), None, i32(0), one, i64(1), one, i64(1), one, None, None, i32(kind), i32(0),
                                  i64(most), i64(1), i64(1), None, ctypes.c_size_t(0), None) == -2


def test_bias_gradient_of_no_input_features_covers_every_row():
    """K = 0 and no activation: db alone is a column sum over all M rows, split like any long sum (a plan that stops after
    its first rows needs no workspace)."""
    L = _native.lib()
    for kind in (0, 1, 2):
        with_inputs = L.smlvm_linear_bwd_workspace_bytes(kind, 0, 1 << 20, 5, 8)
        assert with_inputs > 0 and L.smlvm_linear_bwd_workspace_bytes(kind, 0, 1 << 20, 5, 0) > 0


def test_fuse_linears_leaves_instances_of_their_own():
    """A forward put on the instance (as wrappers of modules do) and hooks on the state dict would be lost without a word."""
    def linear():
        return torch.nn.Linear(3, 3)
    patched, saved, loaded, act = linear(), linear(), linear(), torch.nn.ReLU()
    patched.forward = lambda x: x
    saved.register_state_dict_post_hook(lambda *a: None)
    loaded.register_load_state_dict_post_hook(lambda *a: None)
    act.forward = lambda x: x
    for m in (patched, saved, loaded):
        assert fused.fuse_linears(torch.nn.Sequential(m))[0] is m
    net = fused.fuse_linears(torch.nn.Sequential(linear(), act))
    assert net[0].activation == "none" and net[1] is act
