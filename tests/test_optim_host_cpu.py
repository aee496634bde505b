"""CPU: the host side of the optimiser's operators -- which addresses a call hands over, what a refused call leaves behind (no kernel runs here)."""
import copy
import ctypes as C
import io

import pytest
import torch

from nndetection_amd import _lib as L
from nndetection_amd import optim as O


def stepped(ps, **kw):
    """An AdamW on CPU parameters that has moments of its own and stands at step 5 (from a checkpoint: no kernel involved)."""
    opt = O.AdamW(ps, lr=0.1, **kw)
    opt.load_state_dict({**opt.state_dict(), "state": {i: {"step": 5, "exp_avg": torch.full(p.shape, 1.0 + i), "exp_avg_sq": torch.full(p.shape, 2.0 + i)}
                                                       for i, p in enumerate(ps)}})
    return opt


def recorded(monkeypatch):
    """What the library would have been called with: a list of (name, structs)."""
    calls = []
    monkeypatch.setattr(O, "_run", lambda device, what, words, n, *args: calls.append((what, (L.NndetOptTensor * n).from_buffer_copy(words))))
    return calls


@pytest.mark.parametrize("how", ["deepcopy", "save"])
def test_a_copied_optimizer_steps_its_own_state(monkeypatch, how):
    opt = stepped([torch.nn.Parameter(torch.zeros(4, 5)), torch.nn.Parameter(torch.zeros(7))])
    if how == "deepcopy":
        twin = copy.deepcopy(opt)
    else:
        f = io.BytesIO()
        torch.save(opt, f)
        f.seek(0)
        twin = torch.load(f, weights_only=False)     # (a file that this test wrote)
    calls = recorded(monkeypatch)
    for o in (opt, twin):
        ps = o.param_groups[0]["params"]
        for p in ps:
            p.grad = torch.ones_like(p)
        o.step()
        (what, ts), = calls
        calls.clear()
        state = o.state_dict()["state"]
        assert what == "nndet_adamw_step" and len(ts) == 2
        for i, (t, p) in enumerate(zip(ts, ps)):
            assert (t.param, t.grad, t.numel, t.slot, t.state_bits) == (p.data_ptr(), p.grad.data_ptr(), p.numel(), i, 32)
            assert (t.exp_avg, t.exp_avg_sq) == (state[i]["exp_avg"].data_ptr(), state[i]["exp_avg_sq"].data_ptr())
    assert {t.data_ptr() for st in opt._state.values() for t in st.values()}.isdisjoint(t.data_ptr() for st in twin._state.values() for t in st.values())
