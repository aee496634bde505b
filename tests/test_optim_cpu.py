"""CPU: what the optimiser's operators refuse, their host logic, and the library's own argument checks (no kernel runs here)."""
import ctypes as C
import struct

import pytest
import torch

from nndetection_amd import _lib as L
from nndetection_amd import optim as O


def lists(shapes, dtype=torch.float32):
    p = [torch.zeros(s, dtype=dtype) for s in shapes]
    return p, [torch.zeros_like(x) for x in p], [torch.zeros(s) for s in shapes], [torch.zeros(s) for s in shapes], torch.zeros(len(shapes), dtype=torch.int32)


def refused(match, call):
    with pytest.raises(L.NndetError, match=match):
        call()


@pytest.mark.parametrize("change,match", [
    (lambda a: a[0].append(torch.zeros(3)), "2 grads for 3"),
    (lambda a: a[2].pop(), "1 exp_avgs for 2"),
    (lambda a: a.__setitem__(4, torch.zeros(2)), "steps is one int32"),
    (lambda a: a.__setitem__(4, torch.zeros(1, dtype=torch.int32)), "steps is one int32"),
    (lambda a: a.__setitem__(4, torch.zeros(4, dtype=torch.int32)[::2]), "steps is one int32"),
    (lambda a: a[1].__setitem__(0, torch.zeros(5, 4)), "shape"),
    (lambda a: a[1].__setitem__(0, torch.zeros(4, 5, dtype=torch.float16)), "torch.float16"),
    (lambda a: a[1].__setitem__(0, torch.zeros(4, 5).to_sparse()), "sparse"),
    (lambda a: a[2].__setitem__(0, torch.zeros(5, 4)), "shape"),
    (lambda a: a[2].__setitem__(0, torch.zeros(5, 4).t()), "memory order"),
    (lambda a: a[3].__setitem__(1, torch.zeros(7, dtype=torch.bfloat16)), "bfloat16"),
    (lambda a: a[0].__setitem__(1, torch.zeros(14)[::2]), "not dense"),
    (lambda a: a[0].__setitem__(1, a[0][0]), "shape|twice"),
    (lambda a: a[3].__setitem__(0, a[2][0]), "twice"),
])
def test_adamw_step_refuses(change, match):
    a = list(lists([(4, 5), (7,)]))
    change(a)
    refused(match, lambda: O.adamw_step(*a, lr=1e-3))


def test_adamw_step_refuses_a_duplicate_parameter():
    p, g, m, v, n = lists([(7,), (7,)])
    p[1] = p[0]
    refused("twice", lambda: O.adamw_step(p, g, m, v, n, lr=1e-3))


@pytest.mark.parametrize("kw,match", [
    (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(betas=(0.9, float("nan"))), "betas"), (dict(eps=-1e-8), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=1e-40), "eps"), (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"), (dict(total_norm=torch.zeros(())), "total_norm without"),
    (dict(weight_decay=[0.1]), "1 weight_decay for 2"), (dict(grad_scale=torch.zeros(2)), "grad_scale is one fp32"), (dict(grad_scale=2.0), "grad_scale is one fp32"),
    (dict(found_inf=torch.zeros((), dtype=torch.float64)), "found_inf is one fp32"), (dict(max_norm=1.0, total_norm=torch.zeros(3)), "total_norm is one fp32"),
    (dict(lr=torch.zeros(2)), "lr is one fp32"), (dict(), "no CPU path"),
])
def test_adamw_step_refuses_scalars(kw, match):
    refused(match, lambda: O.adamw_step(*lists([(4, 5), (7,)]), **{"lr": 1e-3, **kw}))


def test_adamw8_and_state_refuse():
    p, g, m, v, n = lists([(300,), (7, 3)])
    ok = O.AdamState8.zeros(p)
    assert [s.numel() for s in ok.exp_avg_scale] == [2, 1] and ok.root[0].dtype == torch.float8_e4m3fn
    step = lambda st: O.adamw8_step(p, g, st, n, lr=1e-3)  # noqa: E731
    refused("no CPU path", lambda: step(ok))
    refused("float8_e4m3fn", lambda: step(ok._replace(exp_avg=m)))
    refused("root_scale", lambda: step(ok._replace(root_scale=[torch.zeros(1), torch.zeros(1)])))
    refused("exp_avg_scale", lambda: step(ok._replace(exp_avg_scale=[torch.zeros(4)[::2], torch.zeros(1)])))
    refused("1 root_scale for 2", lambda: step(ok._replace(root_scale=ok.root_scale[:1])))
    refused("twice", lambda: step(ok._replace(root=ok.exp_avg)))
    for f in (O.write_adam_state8, O.read_adam_state8):
        refused("no CPU path", lambda: f(ok, m, v))
        refused("1 exp_avg_sqs for 2", lambda: f(ok, m, v[:1]))
        refused("torch.float16", lambda: f(ok, [x.half() for x in m], v))
        refused("exp_avg_scale", lambda: f(ok._replace(exp_avg_scale=[torch.zeros(3), torch.zeros(1)]), m, v))
    refused("twice", lambda: O.read_adam_state8(ok, m, m))
    refused("twice", lambda: O.write_adam_state8(ok._replace(root=ok.exp_avg), m, v))
    O.write_adam_state8(O.AdamState8([], [], [], []), [], [])


def test_clip_refuses():
    g = [torch.zeros(4, 5), torch.zeros(7)]
    refused("no CPU path", lambda: O.clip_grads_(g, 1.0))
    refused("no CPU path", lambda: O.grad_norm(g))
    refused("max_norm", lambda: O.clip_grads_(g, -1.0))
    refused("max_norm", lambda: O.clip_grads_(g, float("nan")))
    refused("twice", lambda: O.clip_grads_([g[0], g[0]], 1.0))
    refused("broadcast", lambda: O.clip_grads_([torch.zeros(1).expand(5)], 1.0))
    refused("sparse", lambda: O.clip_grads_([torch.zeros(4, 5).to_sparse()], 1.0))
    refused("float64", lambda: O.clip_grads_([torch.zeros(3, dtype=torch.float64)], 1.0))
    refused("grad_scale", lambda: O.grad_norm(g, torch.zeros(2)))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    refused("norm_type", lambda: O.clip_grad_norm_([p], 1.0, norm_type=1.0))
    refused("no CPU path", lambda: O.clip_grad_norm_(p, 1.0))


def test_dense_and_order():
    x = torch.zeros(2, 3, 4, 5, 6)
    cl = x.contiguous(memory_format=torch.channels_last_3d)
    assert O._dense(x) and O._dense(cl) and O._dense(x.permute(4, 1, 0, 2, 3)) and not O._dense(x[:, 1:]) and not O._dense(x[..., ::2])
    assert not O._dense(torch.zeros(1).expand(4)) and O._dense(torch.zeros(())) and O._dense(torch.zeros(3, 1).t())
    assert not O._same_order(x, cl) and O._same_order(cl, torch.empty_like(cl))
    a, b = torch.zeros(4, 1, 3), torch.zeros(4, 3).unsqueeze(1).as_strided((4, 1, 3), (3, 99, 1))
    assert O._same_order(a, b)


def test_words_are_the_structs():
    wd = struct.unpack("q", struct.pack("d", 0.25))[0]
    w = O._words(2, [11, 21], [12, 22], [13, 23], [14, 24], [15, 25], [16, 26], [17, 27], [wd, wd], [5 | (L.BF16 << 32) | (8 << 48), 6 | (L.F16 << 32) | (32 << 48)])
    assert len(w) == 2 * C.sizeof(L.NndetOptTensor)
    t = (L.NndetOptTensor * 2).from_buffer_copy(w)
    assert (t[1].param, t[1].grad, t[1].exp_avg, t[1].exp_avg_sq, t[1].exp_avg_scale, t[1].root_scale, t[1].numel) == (21, 22, 23, 24, 25, 26, 27)
    assert t[0].weight_decay == 0.25 and (t[0].slot, t[0].dtype, t[0].state_bits) == (5, L.BF16, 8) and (t[1].slot, t[1].dtype, t[1].state_bits) == (6, L.F16, 32)


def test_the_library_checks_its_arguments():
    """Every call below ends before a launch (there may be no GPU here)."""
    lib = L.load()
    one = (L.NndetOptTensor * 1)()
    t = one[0]
    a = L.NndetAdamw(1e-3, 0.9, 0.999, 1e-8, -1.0)
    ws = (C.c_char * (1 << 18))()
    at = (C.addressof(ws) + 15) // 16 * 16
    size = 1 << 17

    def step(n=1, ws=at, size=size, args=a, tensors=one):
        return lib.nndet_adamw_step(tensors, n, C.byref(args) if args is not None else None, ws, size, None)

    t.param = t.grad = t.exp_avg = t.exp_avg_sq = 16
    t.numel, t.state_bits = 4, 32
    assert step(args=None) == -1 and step() == -1                       # no arguments, no steps
    a.steps = 16
    assert step(n=-1) == -1 and step(tensors=None) == -1 and step(ws=None) == -1 and step(ws=at + 4) == -1 and step(size=64) == -2
    for field, bad in (("dtype", 3), ("dtype", -1), ("state_bits", 16), ("numel", -1), ("numel", 1 << 40), ("slot", -1), ("slot", 1 << 24), ("param", 0),
                       ("grad", 0), ("grad", 1 << 48), ("exp_avg", 0), ("exp_avg_sq", 0), ("state_bits", 8)):
        old = getattr(t, field)
        setattr(t, field, bad)
        assert step() == -1, field
        setattr(t, field, old)
    for field, bad in (("beta1", 1.0), ("beta2", -0.5), ("beta2", float("nan")), ("eps", -1.0), ("eps", 1e-40), ("max_norm", float("nan")), ("norm_given", 1)):
        old = getattr(a, field)
        setattr(a, field, bad)
        assert step() == -1, field
        setattr(a, field, old)
    clip = lambda norm, scale, out: lib.nndet_grad_clip(one, 1, norm, scale, out, at, size, None)  # noqa: E731
    assert clip(float("nan"), None, 16) == -1 and clip(1.0, None, None) == -1 and clip(1.0, 16, 16) == -1
    assert lib.nndet_adam_state8(one, 1, 1, at, size, None) == -1       # 32-bit moments
    assert lib.nndet_opt_workspace_bytes(-1) == 0 and lib.nndet_opt_workspace_bytes(2) > lib.nndet_opt_workspace_bytes(1) > 0


def test_the_library_refuses_a_norm_that_is_one_of_its_inputs():
    lib = L.load()
    one = (L.NndetOptTensor * 1)()
    one[0].param = one[0].grad = one[0].exp_avg = one[0].exp_avg_sq = 16
    one[0].numel, one[0].state_bits = 4, 32
    ws = (C.c_char * (1 << 18))()
    for field in ("grad_scale", "lr_device", "found_inf"):
        a = L.NndetAdamw(1e-3, 0.9, 0.999, 1e-8, 1.0)
        a.steps, a.norm = 16, 32
        setattr(a, field, 32)
        assert lib.nndet_adamw_step(one, 1, C.byref(a), (C.addressof(ws) + 15) // 16 * 16, 1 << 17, None) == -1, field


def test_optimizer_refuses():
    p = [torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(3))]
    for kw, match in ((dict(state_bits=16), "state_bits"), (dict(max_norm=-1.0), "max_norm"), (dict(weight_decay=-0.1), "weight_decay"), (dict(betas=(0.9, 1.0)), "betas"),
                      (dict(eps=float("nan")), "eps")):
        refused(match, lambda: O.AdamW(p, **kw))
    refused("twice", lambda: O.AdamW([{"params": p}, {"params": p[:1]}]))
    refused("eps", lambda: O.AdamW([{"params": p, "eps": 1e-42}]))
    refused("amsgrad", lambda: O.AdamW([{"params": p, "amsgrad": True}]))
    refused("float64", lambda: O.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))]))
    opt = O.AdamW(p)
    opt.step()                                                          # no gradients: nothing to do
    p[0].grad = torch.zeros(5)
    refused("no CPU path", opt.step)
    with pytest.raises(ValueError, match="groups"):
        opt.load_state_dict({"state": {}, "param_groups": []})
    refused("bits=8", lambda: opt.state_dict(bits=8))


def test_torch_checkpoint_and_schedule():
    """A checkpoint of torch.optim.AdamW loads into AdamW (fp32 moments: no kernel involved), and back; the schedule reaches the groups."""
    torch.manual_seed(0)
    mk = lambda: [torch.nn.Parameter(torch.randn(4, 3)), torch.nn.Parameter(torch.randn(6)), torch.nn.Parameter(torch.randn(2))]  # noqa: E731
    a, b = mk(), mk()
    ta = torch.optim.AdamW([{"params": a[:2], "weight_decay": 0.1}, {"params": a[2:], "weight_decay": 0.0}], lr=3e-3, betas=(0.8, 0.99), eps=1e-6)
    for _ in range(3):
        for q in a[:2]:
            q.grad = torch.randn_like(q)                                # the last one never gets a gradient: no state
        ta.step()
    o = O.AdamW([{"params": b[:2]}, {"params": b[2:]}])
    o.load_state_dict(ta.state_dict())
    assert o.param_groups[0]["betas"] == (0.8, 0.99) and o.param_groups[0]["eps"] == 1e-6 and o.param_groups[1]["weight_decay"] == 0.0
    sd = o.state_dict()
    assert sorted(sd["state"]) == [0, 1]
    for i in (0, 1):
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(sd["state"][i][k], ta.state_dict()["state"][i][k])
        assert float(sd["state"][i]["step"]) == 3.0
    tb = torch.optim.AdamW([{"params": b[:2]}, {"params": b[2:]}], lr=1.0)
    tb.load_state_dict(sd)
    assert tb.param_groups[0]["lr"] == 3e-3 and tb.param_groups[0]["weight_decay"] == 0.1
    lr = torch.zeros(())
    o2 = O.AdamW([{"params": b[:2]}, {"params": b[2:], "lr": lr}], lr=0.1)
    s = O.LinearWarmupPolyLR(o2, 2, 0.01, 0.9, 10)
    s.step()
    assert o2.param_groups[0]["lr"] == pytest.approx(0.1) and float(lr) == pytest.approx(0.1) and o2.param_groups[1]["lr"] is lr


def test_configure_optimizer_kinds():
    from nndetection_amd.plans import TRAINER_CFG_V001, get_plan
    from nndetection_amd.ptmodule import build_model, configure_optimizer
    m = build_model(get_plan("tiny"))
    for kind, bits in (("adamw", 32), ("adamw8", 8)):
        opt, sched = configure_optimizer(m, dict(TRAINER_CFG_V001, optimizer=kind, max_norm=12.0))
        assert isinstance(opt, O.AdamW) and opt.state_bits == bits and opt.max_norm == 12.0
        assert {g["weight_decay"] for g in opt.param_groups} == {0.0, TRAINER_CFG_V001["weight_decay"]}
        assert opt.param_groups[0]["lr"] == sched.get_lr()
    assert isinstance(configure_optimizer(m, dict(TRAINER_CFG_V001, optimizer="adamw"), lean=False)[0], torch.optim.AdamW)
    assert isinstance(configure_optimizer(m)[0], O.SGDNesterov)
    with pytest.raises(ValueError, match="optimizer"):
        configure_optimizer(m, dict(TRAINER_CFG_V001, optimizer="lion"))
