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


def held(opt):
    return ([(id(p), k, t.data_ptr(), t.clone()) for p, st in opt._state.items() for k, t in st.items()], [(d, t.tolist()) for d, t in opt._steps.items()],
            [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups])


def same(a, b):
    return all(x[:3] == y[:3] and torch.equal(x[3], y[3]) for x, y in zip(a[0], b[0])) and len(a[0]) == len(b[0]) and a[1:] == b[1:]


@pytest.mark.parametrize("change", [
    lambda sd: sd["state"][1].update(exp_avg=torch.zeros(8)), lambda sd: sd["state"][1].update(exp_avg_sq=None), lambda sd: sd["state"][1].pop("exp_avg_sq"),
    lambda sd: sd["state"][1].pop("step"), lambda sd: sd["state"][1].update(step=float("nan")), lambda sd: sd["state"][1].update(step=-1),
    lambda sd: sd["state"][1].update(step=2 ** 31), lambda sd: sd["state"].update({2: sd["state"][1]}), lambda sd: sd["state"].update({-1: sd["state"][1]}),
    lambda sd: sd["state"].update({1: {"step": 1, "exp_avg": torch.zeros(7), "root": torch.zeros(7), "exp_avg_scale": torch.zeros(1), "root_scale": torch.zeros(1)}}),
    lambda sd: sd["state"].update({1: {"step": 1, "exp_avg": torch.zeros(7, dtype=torch.uint8).view(torch.float8_e4m3fn), "exp_avg_scale": torch.zeros(1),
                                       "root": torch.zeros(7, dtype=torch.uint8).view(torch.float8_e4m3fn), "root_scale": torch.zeros(2)}}),
    lambda sd: sd["param_groups"][0].pop("betas"), lambda sd: sd["param_groups"][0].pop("lr"), lambda sd: sd["param_groups"][0].update(betas=(0.9, 1.0)),
    lambda sd: sd["param_groups"][0].update(eps=-1.0), lambda sd: sd["param_groups"][0].update(weight_decay=-1.0), lambda sd: sd["param_groups"][0].update(amsgrad=True),
    lambda sd: sd["param_groups"][0]["params"].pop(),
])
def test_a_refused_checkpoint_changes_nothing(monkeypatch, change):
    """The optimiser goes on as one that was never asked: same moments at the same addresses, counts, groups, and the same next call."""
    opt = stepped([torch.nn.Parameter(torch.zeros(4, 5)), torch.nn.Parameter(torch.zeros(7))])
    bad = copy.deepcopy(opt.state_dict())
    for st in bad["state"].values():
        st["exp_avg"] += 1
        st["step"] += 1
    bad["param_groups"][0].update(lr=0.7, weight_decay=0.3)
    change(bad)
    before = held(opt)
    with pytest.raises((ValueError, L.NndetError)):
        opt.load_state_dict(bad)
    assert same(before, held(opt))
    calls = recorded(monkeypatch)
    for p in opt.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    opt.step()
    assert [(t.exp_avg, t.slot) for t in calls[0][1]] == [(opt._state[p]["exp_avg"].data_ptr(), i) for i, p in enumerate(opt.param_groups[0]["params"])]


def test_versions_of_parameters_that_replays_write(monkeypatch):
    """Outside of a `fresh_params` call every look is another version; within one it is one version, another than before; in a backward pass the last."""
    from nndetection_amd.arch.conv import _pver
    monkeypatch.setattr(L, "graph_written", {})
    net = torch.nn.Linear(3, 2)
    w, b = net.weight, net.bias
    assert _pver(w) == _pver(w)
    L.note_graph_write([w.detach().view(-1)])        # (a view of the parameter: it is the storage that counts)
    seen = [_pver(w) for _ in range(3)]
    assert len(set(seen)) == 3 and _pver(b) == _pver(b)

    class Net(torch.nn.Linear):
        @L.fresh_params
        def inner(self):
            return _pver(w), _pver(w)

        @L.fresh_params
        def forward(self, x):
            return [_pver(w), *self.inner(), _pver(w)]

    outer = Net(3, 2)
    outer.weight, outer.bias = w, b
    first, second = outer(None), outer(None)
    assert len(set(first)) == len(set(second)) == 1 and first[0] != second[0] and first[0] not in seen
    looked = []

    class F(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 1

        @staticmethod
        def backward(ctx, g):
            looked.extend([_pver(w), _pver(w)])
            return g

    F.apply(torch.ones(1, requires_grad=True)).sum().backward()
    assert looked == [second[0]] * 2
    assert _pver(w) != second[0]


def test_requests_that_an_optimiser_cannot_keep_are_refused():
    from nndetection_amd.plans import TRAINER_CFG_V001, get_plan
    from nndetection_amd.ptmodule import RetinaUNetAMDSteps, StandaloneRetinaUNetV001AMD, build_model, configure_optimizer
    m = build_model(get_plan("tiny"))
    for kw, lean, match in ((dict(max_norm=12.0), True, "max_norm"), (dict(max_norm=12.0), False, "max_norm"), (dict(optimizer="adamw", max_norm=1.0), False, "max_norm"),
                            (dict(optimizer="adamw8"), False, "8 bits")):
        with pytest.raises(ValueError, match=match):
            configure_optimizer(m, dict(TRAINER_CFG_V001, **kw), lean=lean)
    assert isinstance(configure_optimizer(m, dict(TRAINER_CFG_V001, max_norm=None), lean=False)[0], torch.optim.SGD)

    class Reference:                                 # (what the registered module inherits from: SGD, whatever the configuration says)
        def configure_optimizers(self):
            return [torch.optim.SGD(self.model.parameters(), 0.1)], []

    class Registered(RetinaUNetAMDSteps, Reference):
        pass

    module = Registered.__new__(Registered)
    module.model = m
    for cfg, ok in ((None, True), ({}, True), (dict(TRAINER_CFG_V001), True), (dict(optimizer="sgd", max_norm=None), True), (dict(optimizer="adamw"), False),
                    (dict(optimizer="adamw8"), False), (dict(max_norm=12.0), False)):
        module.trainer_cfg = cfg
        if ok:
            assert isinstance(module.configure_optimizers()[0][0], torch.optim.SGD)
        else:
            with pytest.raises(ValueError, match="StandaloneRetinaUNetV001AMD"):
                module.configure_optimizers()
    assert StandaloneRetinaUNetV001AMD is not None


def test_the_host_module_is_refused_under_another_torch(monkeypatch):
    assert L.host_lists().built_for.split()[0] == torch.__version__
    monkeypatch.setattr(L, "_host_lists", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(L.NndetError, match="built for torch and Python .* not 1.0.0"):
        L.host_lists()
    assert L._host_lists is None


def test_a_step_without_gradients_has_no_norm():
    opt = stepped([torch.nn.Parameter(torch.zeros(4, 5))], max_norm=1.0)
    opt.grad_norm = torch.tensor(3.0)                # (of an earlier step)
    opt.step()
    assert opt.grad_norm is None


def test_tensors_with_a_negation_to_come(monkeypatch):
    """torch's lazy negation (the imaginary part of a conjugate): a gradient is taken with its sign, what would be written is refused."""
    seen = []
    monkeypatch.setattr(O, "_run", lambda device, what, words, n, *args: seen.append(
        [(C.c_float * t.numel).from_address(t.grad)[:] for t in (L.NndetOptTensor * n).from_buffer_copy(words)]))
    mk = lambda *v: torch._neg_view(torch.tensor(v))  # noqa: E731
    p, m, v, steps = torch.zeros(3), torch.zeros(3), torch.zeros(3), torch.zeros(1, dtype=torch.int32)
    O.adamw_step([p], [mk(1.0, 2.0, 3.0)], [m], [v], steps, lr=0.1)
    O.clip_grads_([mk(1.0, 2.0, 3.0)], 1.0)
    O.grad_norm([mk(4.0, 5.0), torch.conj(torch.complex(torch.zeros(1), torch.ones(1))).imag])
    assert seen == [[[-1.0, -2.0, -3.0]], [[-1.0, -2.0, -3.0]], [[-4.0, -5.0], [-1.0]]]
    g = torch.ones(3)
    for a in (([mk(0.0, 0.0, 0.0)], [g], [m], [v]), ([p], [g], [mk(0.0, 0.0, 0.0)], [v]), ([p], [g], [m], [mk(0.0, 0.0, 0.0)])):
        with pytest.raises(L.NndetError):
            O.adamw_step(*a, steps, lr=0.1)
    with pytest.raises(L.NndetError, match="grad_scale"):
        O.adamw_step([p], [g], [m], [v], steps, lr=0.1, grad_scale=mk(-2.0)[0])
    assert len(seen) == 3


def test_written_states_have_another_version(monkeypatch):
    monkeypatch.setattr(O, "_run", lambda *args: None)
    m, v = [torch.zeros(300)], [torch.zeros(300)]
    st = O.AdamState8.zeros(m)
    codes = [t for ts in st for t in ts]
    count = lambda ts: [t._version for t in ts]  # noqa: E731
    a, b = count(codes), count(m + v)
    O.write_adam_state8(st, m, v)
    assert all(x > y for x, y in zip(count(codes), a)) and count(m + v) == b
    a = count(codes)
    O.read_adam_state8(st, m, v)
    assert all(x > y for x, y in zip(count(m + v), b)) and count(codes) == a


def overlapping(dev):
    """Calls in which one tensor's memory is written for another, and two that are fine: (refused or not, call)."""
    mk = lambda n=300: torch.zeros(n, device=dev)  # noqa: E731
    p, g, m, v, steps = [mk(), mk()], [mk(), mk()], [mk(), mk()], [mk(), mk()], torch.zeros(2, dtype=torch.int32, device=dev)
    st = O.AdamState8.zeros(p)
    one = torch.zeros(2, device=dev)
    params = [torch.nn.Parameter(t) for t in p]
    opt = O.AdamW([{"params": params[:1], "lr": 0.1}, {"params": params[1:], "lr": 0.2}])
    params[0].grad, params[1].grad = g[0], p[0]
    return [("tensor 1 is memory", lambda: O.adamw_step(p, [g[0], p[0]], m, v, steps, lr=0.1)), ("tensor 0 is memory", lambda: O.adamw_step(p, [v[1], g[1]], m, v, steps, lr=0.1)),
            ("twice", lambda: O.adamw8_step(p, g, st._replace(root_scale=st.exp_avg_scale), steps, lr=0.1)),
            ("twice", lambda: O.adamw8_step(p, g, st._replace(root_scale=[one, one]), steps, lr=0.1)),
            ("twice", lambda: O.write_adam_state8(st._replace(exp_avg_scale=[one, one]), m, v)), ("tensor 1 is memory", opt.step),
            (None, lambda: O.adamw_step(p, [g[0], g[0]], m, v, steps, lr=0.1)), (None, lambda: O.adamw_step(p, p, m, v, steps, lr=0.1)),
            (None, lambda: O.read_adam_state8(st._replace(exp_avg_scale=[one, one]), m, v))]


def test_memory_that_is_written_for_another_tensor_is_refused(monkeypatch):
    ran = []
    monkeypatch.setattr(O, "_run", lambda *args: ran.append(args[1]))
    monkeypatch.setattr(O.AdamW, "_init_state", lambda self, p: self._set_state(p, {"exp_avg": torch.zeros(300), "exp_avg_sq": torch.zeros(300)}))
    for match, call in overlapping("cpu"):
        if match:
            with pytest.raises(L.NndetError, match=match):
                call()
        else:
            call()
    assert len(ran) == 3


def test_checkpoints_follow_the_groups_as_they_are():
    """Numbers in a checkpoint run over the groups in order, also after a parameter was moved to another one."""
    ps = [torch.nn.Parameter(torch.zeros(k)) for k in (3, 4, 5)]
    opt = stepped([*ps])
    opt.param_groups.append(dict(opt.param_groups[0], params=[opt.param_groups[0]["params"].pop(0)], weight_decay=0.0))
    sd = copy.deepcopy(opt.state_dict())
    assert [tuple(sd["state"][i]["exp_avg"].shape) for i in range(3)] == [(4,), (5,), (3,)]
    sd["state"][2]["step"] = 9
    opt.load_state_dict(sd)
    assert [float(opt._state[p]["exp_avg"][0]) for p in ps] == [1.0, 2.0, 3.0] and opt._counts(ps[0].device).tolist() == [9, 5, 5]
    opt.param_groups.pop()                           # a parameter that is left out has no number
    assert sorted(opt.state_dict()["state"]) == [0, 1]
    with pytest.raises(ValueError, match="different parameter groups"):
        opt.load_state_dict(sd)


def test_a_module_within_another_ones_call_sees_its_own_replays(monkeypatch):
    """A parameter that is first asked for inside of another module's `fresh_params` call has another version there than before."""
    from nndetection_amd.arch.conv import _pver
    monkeypatch.setattr(L, "graph_written", {})
    w = torch.nn.Parameter(torch.zeros(3))
    L.note_graph_write([w])

    class Inner(torch.nn.Module):
        @L.fresh_params
        def forward(self):
            return _pver(w)

    inner = Inner()

    class Outer(torch.nn.Module):
        @L.fresh_params
        def forward(self):
            return inner(), inner(), _pver(w)

    before, (a, b, c) = inner(), Outer()()
    assert a == b == c != before


def test_lists_of_a_derived_class(monkeypatch):
    ran = []
    monkeypatch.setattr(O, "_run", lambda *args: ran.append(args[1]))

    class Mine(list):
        pass

    p, g, m, v = (Mine([torch.zeros(3)]) for _ in range(4))
    O.adamw_step(p, g, m, v, torch.zeros(1, dtype=torch.int32), lr=0.1)
    O.clip_grads_(g, 1.0)
    st = O.AdamState8(*(Mine(x) for x in O.AdamState8.zeros(m)))
    O.write_adam_state8(st, m, v)
    O.read_adam_state8(st, m, v)
    assert len(ran) == 4


def test_clipping_of_a_strided_leaf_that_requires_a_gradient(monkeypatch):
    """Written back as it was computed, without a word to autograd: like the dense ones, and like torch's clipping."""
    def scale(device, what, words, n, *args):
        for t in (L.NndetOptTensor * n).from_buffer_copy(words):
            (C.c_float * t.numel).from_address(t.grad)[:] = [3.0] * t.numel

    monkeypatch.setattr(O, "_run", scale)
    g = torch.zeros(4, 6)[:, ::2].requires_grad_()
    O.clip_grads_([g], 1.0)
    assert bool((g == 3).all()) and g.is_leaf
