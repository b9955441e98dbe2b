"""CPU: what optim.AdamW and its C entry refuse, before anything touches a GPU."""
import ctypes

import pytest
import torch

from lvmhelpers import _native, optim


def _p(*shape, dtype=torch.float32):
    return torch.nn.Parameter(torch.zeros(*shape, dtype=dtype))


@pytest.mark.parametrize("kwargs", [{"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8},
                                    {"weight_decay": -1.0}, {"state_bits": 16}, {"lr": torch.zeros(2)},
                                    {"lr": torch.zeros((), dtype=torch.float64)}])
def test_bad_hyper_parameters(kwargs):
    with pytest.raises(ValueError):
        optim.AdamW([_p(3)], **kwargs)


def test_bad_parameters_and_gradients():
    with pytest.raises(TypeError):
        optim.AdamW([_p(3, dtype=torch.float64)])
    opt = optim.AdamW([_p(3)])
    with pytest.raises(ValueError):
        opt.step(grads=[])
    with pytest.raises(_native.NativeError):       # no CPU fallback
        opt.step(grads=[torch.zeros(3)])
    with pytest.raises(ValueError):                # torch's own check: the same parameter twice
        p = _p(3)
        optim.AdamW([{"params": [p]}, {"params": [p]}])


def test_state_is_not_made_inside_a_capture(monkeypatch):
    p = _p(3)
    opt = optim.AdamW([p])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError):
        opt._init_state(p, opt.param_groups[0])


def test_a_copied_optimiser_knows_its_parameters():
    import copy
    opt = copy.deepcopy(optim.AdamW([_p(3), _p(4)], state_bits=8))
    assert [opt._order[p] for p in opt.param_groups[0]["params"]] == [0, 1] and opt._tickets == {}


def test_c_entry_checks_its_arguments():
    L = _native.lib()
    d, f, i32 = ctypes.c_double, ctypes.c_float, ctypes.c_int32

    def call(entry, count=1, p=0, g=0, bits=32, b1=0.9, b2=0.999, ticket=16):
        return L.smlvm_adamw_step(ctypes.c_char_p(entry), i32(count), i32(p), i32(g), i32(bits), d(b1), d(b2), f(1e-8),
                                  f(1e-3), None, f(0.0), ctypes.c_uint32(0), ctypes.c_void_p(ticket), None)
    pack = _native.ADAMW_ENTRY.pack
    good = pack(16, 16, 16, 16, 16, 16, 16, 0, 0)                   # n = 0: nothing is launched
    assert call(good) == 0 and call(None, count=0) == 0
    assert call(good, count=-1) == -1 and call(good, p=3) == -1 and call(good, g=-1) == -1
    assert call(good, bits=16) == -1 and call(good, b1=1.0) == -1 and call(good, b2=float("nan")) == -1
    assert call(good, ticket=0) == -1 and call(None) == -1
    for k in (0, 1, 2, 3, 6):
        fields = [16, 16, 16, 16, 16, 16, 16, 5, 0]
        fields[k] = 0
        assert call(pack(*fields)) == -1
    assert call(pack(16, 16, 16, 16, 0, 16, 16, 5, 0), bits=8) == -1
    assert call(pack(16, 16, 16, 16, 0, 0, 16, (1 << 40) + 1, 0)) == -2
    assert call(pack(16, 16, 16, 16, 0, 0, 16, (1 << 64) - 1, 0)) == -1       # n = -1


def test_a_tensor_of_too_many_workgroups_is_refused():
    L = _native.lib()
    d, f, i32 = ctypes.c_double, ctypes.c_float, ctypes.c_int32
    for bits in (32, 8):
        entry = _native.ADAMW_ENTRY.pack(16, 16, 16, 16, 16, 16, 16, 1 << 35, 0)      # 2^24 workgroups of 256 threads
        assert L.smlvm_adamw_step(ctypes.c_char_p(entry), i32(1), i32(0), i32(0), i32(bits), d(0.9), d(0.999), f(1e-8),
                                  f(1e-3), None, f(0.0), ctypes.c_uint32(0), ctypes.c_void_p(16), None) == -2


def test_load_state_dict_keeps_the_kernels_counter_words():
    opt, word = optim.AdamW([_p(3)]), torch.zeros(1, dtype=torch.int32)
    opt._tickets["here"] = word
    opt.load_state_dict(optim.AdamW([_p(3)]).state_dict())
    assert opt._tickets["here"] is word
