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


def _with_state(lr=1e-3, n=4, bits=32):
    """An optimiser on the CPU with a state written by hand, as a step on the GPU would have left it."""
    p = _p(n)
    opt = optim.AdamW([p], lr=lr, state_bits=bits, min_8bit_size=1)
    opt._init_state(p, opt.param_groups[0])
    for k, v in opt.state[p].items():
        v.copy_(torch.arange(v.numel()).view(v.shape) + 1)
    return opt, p


@pytest.fixture
def not_capturing(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def test_load_state_dict_keeps_the_memory_of_rates_and_states(not_capturing):
    rate = torch.tensor(1e-3)
    opt, p = _with_state(rate)
    other, q = _with_state(torch.tensor(5e-4))
    held = dict(opt.state[p])
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] is rate and float(rate) == float(torch.tensor(5e-4))
    assert all(opt.state[p][k] is held[k] for k in held) and other.param_groups[0]["lr"] is not rate
    opt.load_state_dict(_with_state(0.25)[0].state_dict())             # a number fills the tensor
    assert opt.param_groups[0]["lr"] is rate and float(rate) == 0.25
    number, _ = _with_state(0.5)
    number.load_state_dict(other.state_dict())                         # a tensor takes a number's place
    assert float(number.param_groups[0]["lr"]) == float(torch.tensor(5e-4))


def test_load_state_dict_after_a_capture(not_capturing):
    """What the graph writes is not given back: a state that is not loaded starts anew where it is, one of another kind
    is refused before anything changes."""
    opt, p = _with_state()
    held = dict(opt.state[p])
    opt._captured = True
    eight, _ = _with_state(bits=8, lr=0.5)
    with pytest.raises(ValueError):
        opt.load_state_dict(eight.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-3 and opt.param_groups[0]["state_bits"] == 32
    assert all(opt.state[p][k] is v and bool((v != 0).all()) for k, v in held.items())
    opt.load_state_dict(optim.AdamW([_p(4)]).state_dict())
    assert all(opt.state[p][k] is v and bool((v == 0).all()) for k, v in held.items())
    free, q = _with_state()                                            # nothing captured: as the base class
    free.load_state_dict(eight.state_dict())
    assert "exp_rms" in free.state[q]
    free.load_state_dict(optim.AdamW([_p(4)]).state_dict())
    assert not free.state[q]


def test_groups_that_share_a_tensor_rate_load_one_rate(not_capturing):
    def two(a, b):
        return optim.AdamW([{"params": [_p(3)], "lr": a}, {"params": [_p(4)], "lr": b}])
    rate = torch.tensor(1e-3)
    opt = two(rate, rate)
    opt.load_state_dict(two(0.5, 0.5).state_dict())
    assert float(rate) == 0.5
    with pytest.raises(ValueError):
        opt.load_state_dict(two(0.5, 0.25).state_dict())
    assert float(rate) == 0.5 and all(g["lr"] is rate for g in opt.param_groups)


@pytest.mark.parametrize("rate,error", [(torch.tensor(1e-3, dtype=torch.float64), TypeError), (torch.tensor(1e-3).bfloat16(), TypeError),
                                        (torch.tensor(1), TypeError), (torch.full((2,), 1e-3), ValueError),
                                        (torch.empty(0), ValueError)])
def test_a_tensor_rate_is_checked_at_every_step(rate, error):
    """One that took the place of the first rate, by hand or from a checkpoint."""
    opt = optim.AdamW([_p(3)], lr=1e-3)
    opt.step()                                     # (no gradients: nothing to do)
    opt.param_groups[0]["lr"] = rate
    with pytest.raises(error):
        opt.step()
    opt.param_groups[0]["lr"] = torch.tensor([1e-3])
    opt.step()


@pytest.mark.filterwarnings("ignore:optimizer contains")
def test_a_parameter_twice_in_a_group_is_refused():
    """Two entries of one launch would update the same memory at the same time (torch only warns)."""
    p = _p(3)
    with pytest.raises(ValueError):
        optim.AdamW([p, _p(4), p])
    opt = optim.AdamW([_p(4)])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [p, p]})
    assert len(opt.param_groups) == 1


def test_load_state_dict_hooks_see_and_change_what_is_loaded(not_capturing):
    """A hook's own dict is what is loaded, states included, and hooks that run afterwards see them as they stay."""
    opt, p = _with_state(bits=8)
    other, _ = _with_state(bits=8)

    def doubled(opt, sd):
        state = {i: {k: torch.full_like(v, 2) for k, v in st.items()} for i, st in sd["state"].items()}
        return {"state": state, "param_groups": [dict(g, lr=0.125) for g in sd["param_groups"]]}
    seen = {}
    opt.register_load_state_dict_pre_hook(doubled)
    opt.register_load_state_dict_post_hook(lambda o: seen.update({k: (v.dtype, v.clone()) for k, v in o.state[p].items()}))
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] == 0.125 and len(opt._optimizer_load_state_dict_pre_hooks) == 1
    for k, v in opt.state[p].items():
        assert bool((v.float() == 2).all()) and seen[k][0] == v.dtype == other.state_dict()["state"][0][k].dtype
        assert torch.equal(seen[k][1].float(), v.float())
    opt._captured = True
    number, _ = _with_state(bits=32)
    opt.register_load_state_dict_pre_hook(lambda o, sd: number.state_dict())
    with pytest.raises(ValueError):                 # what the hook makes of it is what is checked
        opt.load_state_dict(other.state_dict())
    assert len(opt._optimizer_load_state_dict_pre_hooks) == 2 and bool((opt.state[p]["exp_rms"].float() == 2).all())
