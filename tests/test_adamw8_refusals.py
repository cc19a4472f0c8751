"""What the 8-bit AdamW entry points refuse on the host, without a GPU."""
import ctypes
import os

import pytest
import torch

from dion_amd import _lib
from dion_amd.functional import adamw8_update_foreach, state8_blocks, state8_values

f = ctypes.c_float
tab = lambda *v: (ctypes.c_uint64 * len(v))(*v)  # noqa: E731
sizes = lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libdion_hip.so not built in this checkout")
def test_c_entry_points_refuse():
    lib = _lib.load()

    def step(x=64, xd=1, g=64, gd=1, m=64, ms=64, v=64, vs=64, steps=64, n=8):
        return lib.dion_adamw8_step(tab(x), xd, tab(g), gd, tab(m), tab(ms), tab(v), tab(vs), tab(steps), sizes(n), 1, 64, f(.9), f(.9),
                                    f(1e-8), None, f(0), 0, 0, None)

    for kw, needle in (({"xd": 3}, "x_dtype"), ({"gd": 7}, "g_dtype"), ({"x": 0}, "null"), ({"ms": 0}, "null"), ({"vs": 0}, "null"),
                       ({"v": 0}, "null"), ({"steps": 0}, "null"), ({"n": -1}, "negative"), ({"ms": 66}, "aligned"),
                       ({"n": (1 << 34) + 1}, "2^34")):
        assert step(**kw) == -1 and needle in lib.dion_last_error().decode(), kw
    many = tab(*[64] * 49)
    assert lib.dion_adamw8_step(many, 1, many, 1, many, many, many, many, many, sizes(*[8] * 49), 49, 64, f(.9), f(.9), f(1e-8), None,
                                f(0), 0, 0, None) == -1
    assert "shared" in lib.dion_last_error().decode()
    assert lib.dion_adamw_fp32_state_step(None, 5, None, 0, None, None, None, None, 0, None, f(.9), f(.9), f(1e-8), None, f(0), 0,
                                          None) == -1
    assert lib.dion_state8_values(64, 0, 64, 8, 64, 4, None) == -1
    assert lib.dion_state8_values(64, 0, 64, -8, 64, 0, None) == -1
    assert lib.dion_state8_values(None, 0, 64, 8, 64, 0, None) == -1
    assert lib.dion_state8_values(None, 0, None, 0, None, 0, None) == 0


def test_cpu_tensors_and_wrong_lists_are_refused():
    x, step = torch.zeros(300), [torch.zeros(())]
    codes = ([torch.zeros(300, dtype=torch.int8)], [torch.zeros(3)], [torch.zeros(300, dtype=torch.uint8)], [torch.zeros(3)])
    with pytest.raises(RuntimeError, match="no CPU path"):
        adamw8_update_foreach([x], [x], *codes, 0.1, 0.9, 0.95, 0.0, state_steps=step)
    with pytest.raises(ValueError, match="one tensor for every"):
        adamw8_update_foreach([x], [x], *codes, 0.1, 0.9, 0.95, 0.0, state_steps=[])
    with pytest.raises(RuntimeError, match="no CPU path"):
        state8_values(codes[0][0], codes[1][0])
    adamw8_update_foreach([], [], [], [], [], [], 0.1, 0.9, 0.95, 0.0, state_steps=[])
    assert [state8_blocks(n) for n in (0, 1, 128, 129)] == [0, 1, 1, 2]


def test_group_option_is_checked_and_creates_state():
    from dion import Muon

    def make(**kw):
        return Muon([{"params": [torch.nn.Parameter(torch.zeros(8, 8))]},
                     {"params": [torch.nn.Parameter(torch.zeros(130, dtype=torch.bfloat16))], **kw}], lr=0.1)

    for bad in (4, "8", True, 8.5):
        with pytest.raises(ValueError, match="state_bits"):
            make(algorithm="adamw", state_bits=bad)
    for algo in ("lion", "muon"):
        with pytest.raises(ValueError, match="adamw groups"):
            make(algorithm=algo, state_bits=8)
    opt = make(algorithm="adamw", state_bits=8)
    p = opt.param_groups[1]["params"][0]
    assert {k: (v.dtype, tuple(v.shape)) for k, v in opt.state[p].items()} == {
        "momentum": (torch.int8, (130,)), "momentum_scale": (torch.float32, (2,)), "variance": (torch.uint8, (130,)),
        "variance_scale": (torch.float32, (2,)), "step_dev": (torch.float32, ())}
    # a checkpoint keeps codes and scales as they are (torch would cast them to the parameter's bfloat16)
    opt.state[p]["momentum_scale"].fill_(0.1)
    opt.state[p]["momentum"].fill_(-127)
    saved = opt.state_dict()
    other = make(algorithm="adamw", state_bits=8)
    other.load_state_dict(saved)
    q = other.param_groups[1]["params"][0]
    for key, value in opt.state[p].items():
        assert other.state[q][key].dtype == value.dtype and torch.equal(other.state[q][key], value), key
    assert other.state[q]["momentum"].data_ptr() != opt.state[p]["momentum"].data_ptr()
    saved["state"][1]["variance"] = saved["state"][1]["variance"].float()
    with pytest.raises(ValueError, match="variance"):
        make(algorithm="adamw", state_bits=8).load_state_dict(saved)
    plain = make(algorithm="adamw")
    assert plain.state[plain.param_groups[1]["params"][0]]["momentum"].dtype == torch.bfloat16


def test_group_option_stays_what_it_was():
    from dion import Muon

    p = torch.nn.Parameter(torch.zeros(130, dtype=torch.bfloat16))
    for before, after in ((None, 8), (None, 32), (8, 32), (32, 8)):
        option = {} if before is None else {"state_bits": before}
        opt = Muon([{"params": [p], "algorithm": "adamw", **option}], lr=0.1)
        opt.param_groups[0]["state_bits"] = after
        with pytest.raises(ValueError, match="moments are"):
            opt._adamw_state(p, after)


def test_a_refused_group_is_not_added():
    from dion import Muon

    opt = Muon([torch.nn.Parameter(torch.zeros(8, 8))], lr=0.1)
    for kw in ({"algorithm": "adamw", "state_bits": 16}, {"state_bits": 8}):
        with pytest.raises(ValueError, match="state_bits"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(8))], **kw})
    assert len(opt.param_groups) == 1
    p = torch.nn.Parameter(torch.zeros(8))
    opt.add_param_group({"params": [p], "algorithm": "adamw", "state_bits": 8})
    assert opt.state[p]["momentum"].dtype == torch.int8
