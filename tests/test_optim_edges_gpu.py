"""GPU: calls of the optimiser's operators at the edges of what they accept: second moments below the normal range, tensor counts around the
limits of every launch, steps that are replayed, state that is copied."""
import math

import pytest
import torch

from nndetection_amd import _lib as L
from nndetection_amd import optim as O
from tests.test_optim_gpu import BLOCK, DEV, U, check8, formula, gen, guards_intact, make, rows, within, test_norm_and_clip as norm_and_clip

pytestmark = pytest.mark.gpu
TINY = 2.0 ** -149                                   # one denormal step


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -126, 1e-24, 1e-8])
@pytest.mark.parametrize("sizes", [[300, 1, 257], [70001, 5000, 300]])
def test_second_moments_below_the_normal_range(bits, eps, sizes):
    """Gradients of 2e-20 .. 3e-18: their squares times (1 - b2) are denormal (4e-43 .. 9e-39), the first step is about lr all the same, and so is
    the second from the moments that the first has stored.

    Beside `formula`'s roundings, which are relative, a denormal v is off by half a step of 2^-149 for each operation that makes it (square, two
    products, sum, and with 8 bits the square of the stored root): ev <= 6.06 u v (9.09 with 8 bits) + 2.5 steps. Here v >= 285 steps at the first step, so ev / v
    <= 0.9 %; at the second v is at least 0.999 of that (32 bits), or of the squared least stored root (a code is at most 1/2 below its value
    where codes are denormal: v >= 70 steps, ev / v <= 3.6 %). The root is off by at most ev / v of itself (half, and second order), and
    so is the quotient by at most ev / v / (1 - ev / v)."""
    g = gen(5)
    p = [torch.randn(n, generator=g, device=DEV) for n in sizes]
    gr = [torch.exp2(torch.empty(n, device=DEV).uniform_(-65.4, -58.2, generator=g)) * torch.where(torch.rand(n, generator=g, device=DEV) < 0.5, -1.0, 1.0) for n in sizes]
    steps = torch.zeros(len(sizes), dtype=torch.int32, device=DEV)
    st = O.AdamState8.zeros(p)
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    for t in (1, 2):
        if bits == 8:
            m = [(rows(c.float()).double() * s.double().view(-1, 1)).view(-1)[:c.numel()] for c, s in zip(st.exp_avg, st.exp_avg_scale)]
            v = [(rows(c.float()).double() * s.double().view(-1, 1)).square().view(-1)[:c.numel()] for c, s in zip(st.root, st.root_scale)]
        want = [formula(*x, t, 1e-3, 0.9, 0.999, eps, 0.1) for x in zip(p, gr, m, v)]
        if bits == 8:
            O.adamw8_step(p, gr, st, steps, lr=1e-3, eps=eps, weight_decay=0.1)
        else:
            O.adamw_step(p, gr, m, v, steps, lr=1e-3, eps=eps, weight_decay=0.1)
        for i, (wp, wm, wv) in enumerate(want):
            ev = 1.5 * wv[1] + 2.5 * TINY
            off = ev / wv[0]
            assert float(off.max()) < 0.04
            size, unbias = 1e-3 / (1 - 0.9 ** t), 1 / math.sqrt(1 - 0.999 ** t)
            q = wm[0].abs() / (wv[0].sqrt() * unbias + eps)
            within(p[i], wp[0], 1.5 * wp[1] + size * q * off / (1 - off), what=f"p {sizes[i]} step {t}")
            if bits == 8:
                r = wv[0].sqrt()
                check8(st, i, wm[0], 1.5 * wm[1], r, 6 * U * r + r * off, False)
            else:
                within(m[i], *wm)
                within(v[i], wv[0], ev)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_written_after_the_model_left_the_gpu(bits):
    """model.cpu() before saving: the state lies where it lay, and its counts with it; back on the GPU the training goes on."""
    net = torch.nn.Linear(40, 30).to(DEV)
    opt = O.AdamW(net.parameters(), lr=0.1, state_bits=bits, min_8bit_numel=100)
    for p in net.parameters():
        p.grad = torch.ones_like(p)
    for _ in range(3):
        opt.step()
    want = opt.state_dict(bits=32)
    net.cpu()
    got = opt.state_dict(bits=32)
    for i in (0, 1):
        assert float(got["state"][i]["step"]) == 3.0
        assert all(torch.equal(got["state"][i][k], want["state"][i][k]) for k in ("exp_avg", "exp_avg_sq"))
    with pytest.raises(L.NndetError, match="moved"):
        opt.step()
    net.to(DEV)
    opt.step()
    assert float(opt.state_dict()["state"][0]["step"]) == 4.0


@pytest.mark.parametrize("listed", [True, False])
def test_lazily_cloned_tensors_get_memory_of_their_own(listed):
    """torch._lazy_clone shares the storage until one of the two is written: what a call writes must not reach the other. `listed` False: through
    the Python checks (a gradient in another memory order)."""
    g = gen(7)
    mk = lambda: torch.randn(40, 60, generator=g, device=DEV)  # noqa: E731
    first = {k: mk() for k in "pgm"} | {"v": mk().square()}
    kept = {k: t.clone() for k, t in first.items()}
    lazy = {k: torch._lazy_clone(t) for k, t in first.items()}
    grad = lazy["g"] if listed else lazy["g"].t().contiguous().t()
    steps = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = formula(first["p"], first["g"], first["m"], first["v"], 1, 1e-2, 0.9, 0.999, 1e-8, 0.01)
    O.adamw_step([lazy["p"]], [grad], [lazy["m"]], [lazy["v"]], steps, lr=1e-2)
    O.clip_grads_([lazy["g"]], 0.1)
    assert all(torch.equal(first[k], kept[k]) for k in first)
    for k, w in zip("pmv", want):
        within(lazy[k], *w, what=k)
    st = O.AdamState8.zeros([first["p"]])
    m2, v2 = torch._lazy_clone(first["m"]), torch._lazy_clone(first["v"])
    O.write_adam_state8(st, [m2], [v2])
    lazy8 = O.AdamState8(*([torch._lazy_clone(t[0])] for t in st))
    codes = [t[0].view(torch.uint8).clone() for t in st]
    O.adamw8_step([lazy["p"]], [grad], lazy8, steps, lr=1e-2)
    O.read_adam_state8(lazy8, [m2], [v2])
    assert all(torch.equal(t[0].view(torch.uint8), c) for t, c in zip(st, codes)) and torch.equal(first["m"], kept["m"]) and torch.equal(first["v"], kept["v"])


def capture_steps(opt):
    opt.step()                                       # (the first step makes the state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    return graph


def random_grads(params, seed):
    for i, p in enumerate(params):
        p.grad = torch.randn(p.shape, generator=gen(seed + i), device=DEV)


@pytest.mark.parametrize("fast", [True, False])
def test_a_conv_block_follows_replayed_steps(fast):
    """The packed weights of a block used on its own, forward and backward, after each replay: those of a block that keeps none. `fast` False: two rates."""
    from nndetection_amd.arch.conv import ConvInstanceRelu
    torch.manual_seed(0)
    mk = lambda: ConvInstanceRelu(3, 32, 32, 3, padding=1).to(DEV)  # noqa: E731
    block, plain = mk(), mk()
    ps = list(block.parameters())
    opt = O.AdamW(ps if fast else [{"params": ps[:1], "lr": 0.2}, {"params": ps[1:], "lr": 0.1}], lr=0.2)
    random_grads(ps, 3)
    x = torch.randn(2, 32, 8, 8, 8, generator=gen(1), device=DEV)
    up = torch.randn(2, 32, 8, 8, 8, generator=gen(2), device=DEV)

    def both(net):
        z = x.clone().requires_grad_()
        y = net(z)
        gx, = torch.autograd.grad(y, z, up)          # (the parameters' gradients stay what they are)
        return y.detach(), gx

    both(block)
    graph = capture_steps(opt)
    before = both(block)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        plain.load_state_dict(block.state_dict())
        plain._pack_cache.clear()
        got, want = both(block), both(plain)
        for a, b, old in zip(got, want, before):
            # the two run the same kernels on the same weights; only the order of fp64 sums of the norm may differ
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
            assert float((a - old).abs().max()) > 1e-2 * float(b.abs().max())
        before = got
        with torch.no_grad():
            assert float((block(x) - want[0]).abs().max()) <= 1e-5 * float(want[0].abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_detector_in_evaluation_follows_replayed_steps(dtype):
    from nndetection_amd.plans import get_plan
    from nndetection_amd.ptmodule import build_model
    from tests.gpu_util import synth_inputs
    plan = get_plan("tiny")
    torch.manual_seed(0)
    net = build_model(plan).to(DEV).eval()
    x = synth_inputs(plan)[0].to(DEV, dtype)
    opt = O.AdamW(net.parameters(), lr=3e-2)
    random_grads(net.parameters(), 5)
    logits = lambda: torch.cat([t.float().flatten() for t in net(x)[0].values() if isinstance(t, torch.Tensor)])  # noqa: E731
    probs = lambda: net.inference_step(x)["pred_seg"].float()  # noqa: E731
    with torch.no_grad():
        logits(), probs()
        graph = capture_steps(opt)
        old = logits(), probs()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            got = logits(), probs()
            net.train(), net.eval()                  # (drops everything that is kept of the parameters)
            want = logits(), probs()
            tol = 1e-4 if dtype == torch.float32 else 2e-2           # statistics are summed by atomics; 16 bits store their noise
            for a, b, c in zip(got, want, old):
                assert float((a - b).abs().max()) <= tol * float(b.abs().max())
                assert float((a - c).abs().max()) > 3 * tol * float(b.abs().max())
            old = got


def many(n, big=9000):
    """n sizes, most of them small, some empty: at the ends, and around every 256th place (a look-up reads 256 tensors at a time)."""
    sizes = [1 + (37 * i * i) % 600 for i in range(n)]
    for i in range(n):
        if i % 256 in (0, 255) and i % 512 or i % 50 == 7 or i == n - 1:
            sizes[i] = 0
    sizes[3] = big                                   # (not a call of few small tensors)
    sizes[n - 2] = 2500                              # two tiles behind the last round's boundary
    return sizes


@pytest.mark.parametrize("n", [99, 100, 255, 256, 257, 600])
@pytest.mark.parametrize("clip,dtype", [(False, torch.float32), (True, torch.float32), (True, torch.bfloat16)])
def test_a_step_of_many_tensors_of_one_kind(n, clip, dtype):
    """Around what one launch's arguments hold (99), what a round of the tensor look-up reads (256), and several launches. Each tensor has its own count and decay."""
    x = make(many(n), dtype, seed=n)
    steps = torch.arange(n, dtype=torch.int32, device=DEV)
    wd = [0.1 * (i % 4) for i in range(n)]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in x["g"]))
    factor = 0.5 * norm / (norm + 1e-6) if clip else 1.0
    want = [formula(p, g, m, v, i + 1, 3e-3, 0.9, 0.999, 1e-8, wd[i], factor) for i, (p, g, m, v) in enumerate(zip(*(x[k] for k in "pgmv")))]
    got = O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=3e-3, weight_decay=wd, max_norm=0.5 * norm if clip else None)
    assert got is None if not clip else abs(float(got) - norm) <= 2 * U * norm
    assert torch.equal(steps, torch.arange(1, n + 1, dtype=torch.int32, device=DEV))
    for i, (wp, wm, wv) in enumerate(want):          # (clipped: the norm's and the factor's rounding, as in the tests of few tensors)
        within(x["p"][i], wp[0], 1.5 * wp[1], dtype, f"p {i}")
        within(x["m"][i], wm[0], 1.5 * wm[1], what=f"m {i}")
        within(x["v"][i], wv[0], 1.5 * wv[1], what=f"v {i}")
    assert all(guards_intact(v, b, 0) for v, b in x["buf"])


@pytest.mark.parametrize("n", [76, 77, 256, 257, 600])
@pytest.mark.parametrize("clip,dtype", [(False, torch.float32), (True, torch.float32), (True, torch.float16)])
def test_an_8_bit_step_of_many_tensors_of_one_kind(n, clip, dtype):
    """The same with 8-bit moments (76 tensors a launch), written and read back on the way."""
    sizes = many(n)
    x = make(sizes, dtype, seed=1000 + n)
    st = O.AdamState8.zeros(x["p"])
    O.write_adam_state8(st, x["m"], x["v"])
    for i, k in enumerate(sizes):
        if k:
            r = x["v"][i].double().sqrt()
            check8(st, i, x["m"][i].double(), torch.zeros_like(r), r, U * r + TINY, True)
    m0, v0 = [torch.empty_like(t) for t in x["m"]], [torch.empty_like(t) for t in x["v"]]
    O.read_adam_state8(st, m0, v0)
    for i, k in enumerate(sizes):
        m = (rows(st.exp_avg[i].float()) * st.exp_avg_scale[i].view(-1, 1)).view(-1)[:k]
        r = (rows(st.root[i].float()) * st.root_scale[i].view(-1, 1)).view(-1)[:k]
        assert torch.equal(m0[i], m) and torch.equal(v0[i], r * r)
    steps = torch.arange(n, dtype=torch.int32, device=DEV)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in x["g"]))
    factor = 0.5 * norm / (norm + 1e-6) if clip else 1.0
    want = [formula(p, g, m, v, i + 1, 3e-3, 0.9, 0.999, 1e-8, 0.1, factor) for i, (p, g, m, v) in enumerate(zip(x["p"], x["g"], m0, v0))]
    got = O.adamw8_step(x["p"], x["g"], st, steps, lr=3e-3, weight_decay=0.1, max_norm=0.5 * norm if clip else None)
    assert got is None if not clip else abs(float(got) - norm) <= 2 * U * norm
    assert torch.equal(steps, torch.arange(1, n + 1, dtype=torch.int32, device=DEV))
    for i, (wp, wm, wv) in enumerate(want):
        if sizes[i]:
            within(x["p"][i], wp[0], 2 * wp[1], dtype, f"p {i}")
            r = wv[0].sqrt()
            check8(st, i, wm[0], 2 * wm[1], r, 8 * U * r + 2.0 ** -74, False)
    assert all(guards_intact(v, b, 0) for v, b in x["buf"])


@pytest.mark.parametrize("n", [164, 165, 256, 257, 600])
@pytest.mark.parametrize("big", [9000, 300])
def test_clipping_of_many_tensors_of_one_type(n, big):
    """Around what one launch's arguments hold (164), with and without the kernel for few small tensors. (test_norm_and_clip adds two tensors.)"""
    for dtype in (torch.float32, torch.bfloat16):
        norm_and_clip(dtype, 1, many(n, big))
        norm_and_clip(dtype, 0, many(n - 2, big))


@pytest.mark.parametrize("clip", [False, True])
def test_an_optimizer_of_both_kinds_of_moments_with_many_tensors(clip):
    """AdamW(state_bits=8) with 120 parameters that keep 32 bits and 90 that do not: two tables of two launches each, two sums and two steps."""
    shapes = [(1 + i % 97,) if i % 7 < 4 else (64, 64 + i % 5) for i in range(210)]
    g = gen(11)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g, device=DEV)) for s in shapes]
    random_grads(ps, 700)
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
    opt = O.AdamW([{"params": ps[::2], "weight_decay": 0.1}, {"params": ps[1::2], "weight_decay": 0.0}], lr=1e-2, state_bits=8, max_norm=0.5 * norm if clip else None)
    factor = 0.5 * norm / (norm + 1e-6) if clip else 1.0
    for t in (1, 2):
        old = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
        if t == 2:
            full = opt.state_dict(bits=32)["state"]
            order = [*range(0, 210, 2), *range(1, 210, 2)]
            for i, st in full.items():
                old[0][order[i]], old[1][order[i]] = st["exp_avg"], st["exp_avg_sq"]
        want = [formula(p.detach(), p.grad, m, v, t, 1e-2, 0.9, 0.999, 1e-8, 0.0 if i % 2 else 0.1, factor) for i, (p, m, v) in enumerate(zip(ps, *old))]
        opt.step()
        for i, (p, w) in enumerate(zip(ps, want)):
            within(p.detach(), w[0][0], 2 * w[0][1], what=f"{i} step {t}")
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    kinds = [("root" in st) for st in opt.state_dict()["state"].values()]
    assert sum(kinds) == 90 and len(kinds) == 210


def test_memory_that_is_written_for_another_tensor_is_refused():
    """Through the fast path too, before anything runs."""
    from tests.test_optim_host_cpu import overlapping
    for match, call in overlapping(DEV):
        if match:
            with pytest.raises(L.NndetError, match=match):
                call()
        else:
            call()


def test_the_second_moment_of_many_8_bit_steps():
    """600 steps at b2 = 0.99 with gradients drawn from four magnitudes: the mean second moment is that of the format's own recursion -- a Markov chain
    over the 127 codes, exact in 64 bits -- and that lies 0 .. 8 % above the mean square of the gradients, which is what 32-bit moments settle at.

    One element of each block has the gradient that keeps it at 448, so every scale stays 1. The mean over n independent elements is off by at most
    6 standard deviations / sqrt(n). The kernel's probabilities are multiples of 2^-16 taken at their middle: a step is off by 2^-17 of a code's distance (at
    most r / 8, i.e. 2^-19 of v), and 1 / (1 - b2) steps add up: 100 * 2^-19 of v."""
    n, b2, N = 256 * 256, 0.99, 600
    sizes = [4.0, 12.0, 20.0, 40.0]
    code = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    T = torch.zeros(127, 127, dtype=torch.float64)
    for a in sizes:
        r = (b2 * code * code + (1 - b2) * a * a).sqrt()
        lo = (torch.searchsorted(code, r, right=True) - 1).clamp(0, 125)
        up = ((r - code[lo]) / (code[lo + 1] - code[lo])).clamp(0, 1)
        assert int(lo.min()) > 0                     # (never near the least code, which has a rule of its own)
        T[torch.arange(127), lo] += (1 - up) / 4
        T[torch.arange(127), lo + 1] += up / 4
    at = torch.zeros(127, dtype=torch.float64)
    at[(code == 24.0).nonzero()] = 1.0               # the start: r = 24, a code
    for _ in range(N):
        at = at @ T
    mean = float(at @ code ** 2)
    var = float(at @ code ** 4) - mean ** 2
    true = sum(a * a for a in sizes) / 4
    assert 1.0 < mean / true < 1.08
    r = torch.full((n,), 24.0, device=DEV)
    r[::BLOCK] = 448.0
    p, st, steps = torch.zeros(n, device=DEV), O.AdamState8.zeros([r]), torch.zeros(1, dtype=torch.int32, device=DEV)
    O.write_adam_state8(st, [torch.zeros(n, device=DEV)], [r * r])
    table, g = torch.tensor(sizes, device=DEV), gen(12)
    for _ in range(N):
        grad = table[torch.randint(0, 4, (n,), generator=g, device=DEV)]
        grad[::BLOCK] = 448.0
        O.adamw8_step([p], [grad], st, steps, lr=0.0, betas=(0.9, b2))
    assert bool((st.root_scale[0] - 1).abs().max() <= N * 4 * U)
    got = rows(st.root[0].float()).double()[:, 1:].square().mean()
    count = 255 * 256
    assert abs(float(got) - mean) <= 6 * math.sqrt(var / count) + 100 * 2.0 ** -19 * mean + N * 16 * U * mean
    assert float(got) > true                         # (the bias that the documentation states is there)


def test_parameters_that_change_their_group():
    """The groups are read at every step: a parameter takes the decay of the group it is in, one that was taken out stays as it is."""
    ps = [torch.nn.Parameter(torch.randn(300, generator=gen(i), device=DEV)) for i in range(3)]
    opt = O.AdamW([{"params": ps[:2], "weight_decay": 0.5}, {"params": ps[2:], "weight_decay": 0.0}], lr=0.1)
    random_grads(ps, 20)
    opt.step()
    a, b = (g["params"] for g in opt.param_groups)
    for change, decays in ((lambda: (b.insert(0, a.pop(1))), (0.5, 0.0, 0.0)), (lambda: (a.append(b.pop(1)), b.append(a.pop(0))), (0.0, 0.0, 0.5)), (lambda: a.pop(0), (0.0, 0.0, None))):
        change()
        old = [p.detach().clone() for p in ps]
        st = {i: {k: v.clone() for k, v in opt._state[p].items()} for i, p in enumerate(ps)}
        t = [int(opt._steps[ps[0].device][i]) + 1 for i in range(3)]
        opt.step()
        for i, (p, wd) in enumerate(zip(ps, decays)):
            if wd is None:
                assert torch.equal(p, old[i])
            else:
                within(p.detach(), *formula(old[i], p.grad, st[i]["exp_avg"], st[i]["exp_avg_sq"], t[i], 0.1, 0.9, 0.999, 1e-8, wd)[0], what=f"{i}")


@pytest.mark.parametrize("clip", [False, True])
def test_three_rates_after_the_first_step(clip):
    """Parameters of one rate scattered over the groups, some without a gradient, a rate whose parameters have none: one call a rate, one norm over all."""
    ps = [torch.nn.Parameter(torch.randn(k, generator=gen(k), device=DEV)) for k in (300, 5, 4097, 64, 1000, 7)]
    lr = torch.tensor(0.05, device=DEV)
    groups = [dict(params=[ps[0], ps[1]], lr=0.1, weight_decay=0.1), dict(params=[ps[2]], lr=lr, weight_decay=0.2), dict(params=[ps[3], ps[4]], lr=0.1, weight_decay=0.0),
              dict(params=[ps[5]], lr=0.3, weight_decay=0.3)]
    rates = [0.1, 0.1, float(lr), 0.1, 0.1, 0.3]
    decays = [0.1, 0.1, 0.2, 0.0, 0.0, 0.3]
    opt = O.AdamW(groups, max_norm=0.5 if clip else None)
    random_grads(ps, 30)
    opt.step()
    for without in ((), (1,), (5,), (0, 1, 3, 4, 5)):
        random_grads(ps, 40 + len(without))
        for i in without:
            ps[i].grad = None
        live = [i for i in range(6) if i not in without]
        norm = math.sqrt(sum(float(ps[i].grad.double().square().sum()) for i in live))
        factor = min(1.0, 0.5 / (norm + 1e-6)) if clip else 1.0
        st = {i: {k: v.clone() for k, v in opt._state[p].items()} for i, p in enumerate(ps)}
        t = opt._steps[ps[0].device].tolist()
        old = [p.detach().clone() for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            if i in without:
                assert torch.equal(p, old[i])
                continue
            wp, _, _ = formula(old[i], p.grad, st[i]["exp_avg"], st[i]["exp_avg_sq"], t[i] + 1, rates[i], 0.9, 0.999, 1e-8, decays[i], factor)
            within(p.detach(), wp[0], 1.5 * wp[1], what=str(i))
        assert opt._steps[ps[0].device].tolist() == [k + (i not in without) for i, k in enumerate(t)]
        assert opt.grad_norm is None if not clip else abs(float(opt.grad_norm) - norm) <= 2 * U * norm


def test_a_tensor_without_storage_leaves_nothing_behind():
    """torch.func's wrappers have no address: the call raises, and frees what it had packed (500 structs of 72 bytes) until then."""
    import tracemalloc
    gs = [torch.zeros(1, device=DEV) for _ in range(500)]

    def call(x):
        with pytest.raises(RuntimeError):
            O.grad_norm([*gs, x])
        return x.sum()

    x = torch.zeros(3, device=DEV)
    torch.func.grad(call)(x)
    tracemalloc.start()
    try:
        before = tracemalloc.get_traced_memory()[0]
        for _ in range(20):
            torch.func.grad(call)(x)
        assert tracemalloc.get_traced_memory()[0] - before < 5 * 72 * 500
    finally:
        tracemalloc.stop()
