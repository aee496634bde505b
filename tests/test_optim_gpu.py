"""GPU: the optimiser's operators against plain implementations in 64 bits.

Tolerances count roundings. u = 2^-24 is half an fp32 step relative to the value. A product of two rounded factors and a sum, as the step makes
them, gives for the moments at most 4 u (|b1 m| + |(1 - b1) g|) and 6 u of the (positive) second moment: constants, the gradient's factor,
products and sum each once. The root halves 6 u and adds its own: 4 u. The denominator adds the constant, the product and the sum: 7 u; the quotient
one more, the step size two. The parameter adds decay (2 u of p) and the difference (u of the result). A type of 16 bits rounds once more, by half
its step. Second-order terms are covered by 1 %."""
import math

import pytest
import torch

from nndetection_amd import _lib as L
from nndetection_amd import optim as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda"
BLOCK = O.STATE8_BLOCK
HALF = {torch.float32: (U, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
SMALL = [1, 2, 3, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 4095, 4096]      # (a call of few small tensors has kernels of its own)
SIZES = SMALL[:-2] + [4097, 70001]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def place(x, shift):
    """x (1-D) at `shift` elements behind an aligned address, with a guard of 9 elements on either side of it."""
    buf = torch.full((x.numel() + 64 + shift,), 7.0, dtype=x.dtype, device=DEV) if x.dtype != torch.float8_e4m3fn else \
        torch.full((x.numel() + 64 + shift,), 7, dtype=torch.uint8, device=DEV).view(x.dtype)
    v = buf[32 + shift:32 + shift + x.numel()]
    v.copy_(x)
    return v, buf


def guards_intact(v, buf, shift):
    b = buf.view(torch.uint8) if buf.dtype == torch.float8_e4m3fn else buf
    return bool((b[:32 + shift] == 7).all()) and bool((b[32 + shift + v.numel():] == 7).all())


def make(sizes, dtype, seed=0, shift=0, zero_every=5):
    g = gen(seed)
    out = {k: [] for k in ("p", "g", "m", "v", "buf")}
    for i, n in enumerate(sizes):
        s = 10.0 ** (-i % 4)
        gr = torch.randn(n, generator=g, device=DEV) * s * (0.0 if i % zero_every == zero_every - 1 else 1.0)
        m = torch.randn(n, generator=g, device=DEV) * s * 0.3
        v = (m * torch.rand(n, generator=g, device=DEV) * 4).square()
        for k, x in (("p", torch.randn(n, generator=g, device=DEV).to(dtype)), ("g", gr.to(dtype)), ("m", m), ("v", v)):
            view, buf = place(x, shift)
            out[k].append(view)
            out["buf"].append((view, buf))
    return out


def formula(p, g, m, v, t, lr, b1, b2, eps, wd, factor=1.0):
    """The step in 64 bits, and how far fp32 may be off: (new, bound) of p (before its own type's rounding), m, v."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * factor
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em, ev = 4.04 * U * (b1 * m.abs() + (1 - b1) * g.abs()), 6.06 * U * v1
    unbias, size = 1 / math.sqrt(1 - b2 ** t), lr / (1 - b1 ** t)
    den = v1.sqrt() * unbias + eps
    q = m1 / den
    new = p * (1 - lr * wd) - size * q
    ep = 2.02 * U * p.abs() + size * (em / den + 10.1 * U * q.abs()) + 1.01 * U * new.abs()
    tiny = 2.0 ** -149                               # one denormal step for products that fall below the normal range
    return (new, ep + tiny), (m1, em + 4 * tiny), (v1, ev + 4 * tiny)


def within(got, want, bound, dtype=torch.float32, what=""):
    rel, least = HALF[dtype]
    bound = bound + (0 if dtype == torch.float32 else rel * (want.abs() + bound) + least)
    off = (got.double() - want).abs()
    worst = float((off - bound).max()) if off.numel() else -1.0
    assert worst <= 0, f"{what}: off by {float(off.max())}, {worst} over the bound"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("t0", [0, 999])
@pytest.mark.parametrize("sizes", [SIZES, SMALL, SMALL[:1]])
def test_adamw_step(dtype, shift, t0, sizes):
    x = make(sizes, dtype, seed=t0 + shift, shift=shift)
    wd = [0.0 if i % 3 == 0 else 0.1 for i in range(len(sizes))]
    steps = torch.full((len(sizes) + 2,), t0, dtype=torch.int32, device=DEV)
    if t0 == 0:
        for m, v in zip(x["m"], x["v"]):
            m.zero_(), v.zero_()
    want = [formula(p, g, m, v, t0 + 1, 3e-3, 0.9, 0.999, 1e-8, w) for p, g, m, v, w in zip(x["p"], x["g"], x["m"], x["v"], wd)]
    grads = [g.clone() for g in x["g"]]
    versions = [p._version for p in x["p"]]
    assert O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=3e-3, weight_decay=wd) is None
    assert steps.tolist() == [t0 + 1] * len(sizes) + [t0, t0]
    for i, (wp, wm, wv) in enumerate(want):
        within(x["p"][i], *wp, dtype, f"p {sizes[i]}")
        within(x["m"][i], *wm, what=f"m {sizes[i]}")
        within(x["v"][i], *wv, what=f"v {sizes[i]}")
        assert torch.equal(x["g"][i], grads[i]) and x["p"][i]._version > versions[i]
    assert all(guards_intact(v, b, shift) for v, b in x["buf"])


def test_adamw_many_tensors_of_mixed_types():
    """300 tensors (several table launches), all three types in one call, empty ones among them."""
    sizes = [(7 * i * i) % 1500 if i % 10 else 0 for i in range(300)]
    types = [torch.float32, torch.bfloat16, torch.float16]
    x = {k: [] for k in "pgmv"}
    for i, n in enumerate(sizes):
        y = make([n], types[i % 3], seed=i)
        for k in "pgmv":
            x[k].append(y[k][0])
    steps = torch.arange(300, dtype=torch.int32, device=DEV)
    want = [formula(p, g, m, v, i + 1, 1e-2, 0.8, 0.95, 1e-6, 0.01) for i, (p, g, m, v) in enumerate(zip(*(x[k] for k in "pgmv")))]
    O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=1e-2, betas=(0.8, 0.95), eps=1e-6)
    assert torch.equal(steps, torch.arange(1, 301, dtype=torch.int32, device=DEV))
    for i, (wp, wm, wv) in enumerate(want):
        within(x["p"][i], *wp, types[i % 3], f"p {i}")
        within(x["m"][i], *wm)
        within(x["v"][i], *wv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9, math.inf])
@pytest.mark.parametrize("more", [0, 70000])
def test_adamw_clip_and_scale(dtype, max_norm, more):
    """The norm is of the unscaled gradients; its factor and the scale's are one fp32 number (half a step more than `formula` counts: 6.06 -> 8.08
    of v and 4.04 -> 5.05 of m would do; the factor's rounding is in the counts already, the norm's own is one more)."""
    x = make([5, 300, 2048 + more, 1111], dtype, seed=3)
    scale = torch.tensor(48.0, device=DEV)
    g64 = [g.double() / 48.0 for g in x["g"]]
    norm = math.sqrt(sum(float(g.square().sum()) for g in g64))
    factor = min(1.0, max_norm / (norm + 1e-6)) / 48.0
    steps = torch.full((4,), 10, dtype=torch.int32, device=DEV)
    want = [formula(p, g, m, v, 11, 1e-2, 0.9, 0.999, 1e-8, 0.0, factor) for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"])]
    got = O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=1e-2, weight_decay=0.0, max_norm=max_norm, grad_scale=scale,
                       found_inf=torch.zeros((), device=DEV))
    assert abs(float(got) - norm) <= 2 * U * norm
    for i, (wp, wm, wv) in enumerate(want):
        within(x["p"][i], wp[0], 1.5 * wp[1], dtype)
        within(x["m"][i], wm[0], 1.5 * wm[1])
        within(x["v"][i], wv[0], 1.5 * wv[1])


def test_adamw_given_norm_and_rate_on_the_device():
    x = make([700, 33], torch.float32, seed=4)
    steps = torch.zeros(2, dtype=torch.int32, device=DEV)
    lr = 0.0123
    want = [formula(p, g, m, v, 1, float(torch.tensor(lr)), 0.9, 0.999, 1e-8, 0.01, 1.0 / (4.0 + 1e-6)) for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"])]
    total = torch.tensor([4.0], device=DEV)
    assert O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=torch.tensor(lr, device=DEV), max_norm=1.0, total_norm=total) is total
    assert float(total) == 4.0
    for i, (wp, wm, wv) in enumerate(want):
        within(x["p"][i], *wp)
        within(x["m"][i], *wm)
        within(x["v"][i], *wv)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("flag", [1.0, math.inf, math.nan])
@pytest.mark.parametrize("most", [4000, 5000])
def test_a_skipped_step_changes_nothing(bits, flag, most):
    x = make([700, 33, most], torch.float32, seed=5)
    x["g"][1][3] = math.inf
    steps = torch.full((3,), 6, dtype=torch.int32, device=DEV)
    st = O.AdamState8.zeros(x["p"])
    O.write_adam_state8(st, x["m"], x["v"])
    held = [t for k in "pmv" for t in x[k]] + [steps] + [t.view(torch.uint8) for k in st for t in k]
    before = [t.clone() for t in held]
    kw = dict(lr=0.1, found_inf=torch.tensor(flag, device=DEV), grad_scale=torch.tensor(2.0, device=DEV), max_norm=1.0)
    norm = O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, **kw) if bits == 32 else O.adamw8_step(x["p"], x["g"], st, steps, **kw)
    assert math.isinf(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(held, before))


def test_missing_gradients_and_memory_orders():
    """grads None: untouched; parameters in channels-last order; gradients in another order, expanded, sliced; scalars."""
    g = gen(6)
    w = torch.randn(6, 4, 3, 3, 3, generator=g, device=DEV)
    p = [w.contiguous(memory_format=torch.channels_last_3d), w.clone(), torch.randn(5, 7, generator=g, device=DEV).t(), torch.randn((), generator=g, device=DEV),
         torch.randn(9, generator=g, device=DEV), torch.randn(8, 3, generator=g, device=DEV)]
    r = torch.randn(6, 4, 3, 3, 3, generator=g, device=DEV)
    gr = [r.clone(), r.contiguous(memory_format=torch.channels_last_3d), torch.randn(7, 5, generator=g, device=DEV), torch.full((), 2.0, device=DEV), None,
          torch.randn(8, 6, generator=g, device=DEV)[:, ::2]]
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    steps = torch.zeros(6, dtype=torch.int32, device=DEV)
    want = [formula(a, b, c, d, 1, 1e-2, 0.9, 0.999, 1e-8, 0.01) for a, b, c, d in zip(p, [b if b is not None else torch.zeros(9, device=DEV) for b in gr], m, v)]
    kept = p[4].clone()
    O.adamw_step(p, gr, m, v, steps, lr=1e-2)
    for i in (0, 1, 2, 3, 5):
        within(p[i], *want[i][0], what=str(i))
        within(m[i], *want[i][1], what=str(i))
    assert torch.equal(p[4], kept) and not m[4].any() and steps.tolist() == [1, 1, 1, 1, 0, 1]
    assert p[0].is_contiguous(memory_format=torch.channels_last_3d)
    O.adamw_step([p[0]], [torch.ones(1, device=DEV).expand(p[0].shape)], [m[0]], [v[0]], steps[:1], lr=0.0, weight_decay=0.0)
    assert int(steps[0]) == 2
    assert O.adamw_step([], [], [], [], steps, lr=0.1, max_norm=1.0).item() == 0.0
    assert O.adamw_step([p[4]], [None], [m[4]], [v[4]], steps, lr=0.1) is None


def test_not_finite_gradients_stay_where_they_are():
    """Without a scaler's flag an inf or NaN reaches its own element (fp32 moments), as in the formula."""
    x = make([600], torch.float32, seed=7)
    x["g"][0][5], x["g"][0][300] = math.nan, math.inf
    steps = torch.zeros(1, dtype=torch.int32, device=DEV)
    O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=0.1)
    bad = torch.zeros(600, dtype=torch.bool, device=DEV)
    bad[5] = bad[300] = True
    assert torch.equal(~torch.isfinite(x["p"][0]), bad) and torch.equal(~torch.isfinite(x["m"][0]), bad)


# ---- 8 bits

def mix(pair, t):
    """The documented bits, in Python's whole numbers."""
    m = 0xFFFFFFFF
    x = (pair + t * 0x9E3779B1) & m
    x = ((x ^ (x >> 16)) * 0x6A09E667) & m
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & m
    return x ^ (x >> 16)


def rows(x):
    """1-D to blocks of 256, zeros behind the last element."""
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def step8(x, codes, scale):
    """Distance between e4m3 neighbours around |x|, in units of x: the bound of a rounding up or down (half of it: to nearest)."""
    e = torch.floor(torch.log2((x.abs() / scale.clamp_min(2.0 ** -126)).clamp_min(2.0 ** -6)))
    return torch.exp2(e - 3) * scale


def check8(st, i, m, em, r, er, nearest):
    """The state's moments are the ones wanted (m, r = sqrt v in 64 bits, with their fp32 bounds) to a rounding of e4m3; scales are the blocks' maxima."""
    for name, codes, scale, want, bound in (("m", st.exp_avg[i], st.exp_avg_scale[i], m, em), ("r", st.root[i], st.root_scale[i], r, er)):
        w, b, c, s = rows(want), rows(bound), rows(codes.float()), scale.double().view(-1, 1)
        top = w.abs().amax(1, keepdim=True)
        assert bool(((s - top / 448).abs() <= (3 * U * top + b.amax(1, keepdim=True)) / 448 + 2.0 ** -149).all()), name
        part = 0.5 if name == "m" or nearest else 1.0
        # a code below one step of the format: a root that is not 0 is kept off 0 (one whole step of 2^-9)
        least = torch.where((w > 0) & (name == "r"), 2.0 ** -9 * s, torch.zeros_like(s))
        allowed = torch.maximum(part * step8(w, c, s) * (1 + 8 * U), least) + 2 * b + 4 * U * w.abs()
        off = (c.double() * s - w).abs() - allowed
        assert float(off.max()) <= 0, f"{name}: {float(off.max())} over the bound"
        if name == "r":
            assert bool((c[w > 2.0 ** -70] > 0).all()), "a root that is not zero was stored as zero"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("t0", [0, 777])
@pytest.mark.parametrize("sizes", [SIZES, SMALL])
def test_adamw8_step(dtype, shift, t0, sizes):
    x = make(sizes, dtype, seed=10 + t0 + shift, shift=shift)
    st = O.AdamState8(*([] for _ in range(4)))
    bufs = []
    for z in O.AdamState8.zeros(x["p"])._asdict().items():
        for t in z[1]:
            v, b = place(t.reshape(-1), shift if t.dtype == torch.float8_e4m3fn else 0)
            getattr(st, z[0]).append(v)
            bufs.append((v, b))
    if t0:
        O.write_adam_state8(st, x["m"], x["v"])
    m0 = [(rows(c.float()).double() * s.double().view(-1, 1)).view(-1)[:c.numel()] for c, s in zip(st.exp_avg, st.exp_avg_scale)]
    r0 = [(rows(c.float()).double() * s.double().view(-1, 1)).view(-1)[:c.numel()] for c, s in zip(st.root, st.root_scale)]
    steps = torch.full((len(sizes),), t0, dtype=torch.int32, device=DEV)
    want = [formula(p, g, m, r * r, t0 + 1, 3e-3, 0.9, 0.999, 1e-8, 0.1) for p, g, m, r in zip(x["p"], x["g"], m0, r0)]
    O.adamw8_step(x["p"], x["g"], st, steps, lr=3e-3, weight_decay=0.1)
    assert steps.tolist() == [t0 + 1] * len(sizes)
    for i, (wp, wm, wv) in enumerate(want):
        # two more roundings than `formula` counts: the decoded moments' products (m: 1 u; v: 3 u)
        within(x["p"][i], wp[0], 1.5 * wp[1], dtype, f"p {sizes[i]}")
        r = wv[0].sqrt()
        check8(st, i, wm[0], 1.5 * wm[1], r, 6 * U * r + 2.0 ** -74, False)
    assert all(guards_intact(v, b, shift if v.dtype == torch.float8_e4m3fn else 0) for v, b in bufs)


def plain8(m, r, t):
    """Codes and scales of a step in fp32 on the CPU, operation by operation as documented (every one an IEEE operation)."""
    out = []
    for x, root in ((rows(m.cpu()), False), (rows(r.cpu()), True)):
        s = x.abs().amax(1, keepdim=True) * torch.tensor(1.0 / 448.0)
        s = torch.where(s < 2.0 ** -110, torch.zeros_like(s), s)
        y = torch.where(s > 0, x * (1.0 / s), torch.zeros_like(x))
        if not root:
            out += [y.to(torch.float8_e4m3fn).view(torch.uint8), s.view(-1)]
            continue
        n = x.numel()
        bits = torch.tensor([mix(i, t) for i in range(n // 2)], dtype=torch.int64)
        u = torch.stack([bits & 0xFFFF, bits >> 16], 1).view(x.shape) * 16 + 8
        c = (((y * 2.0 ** -120).view(torch.int32).long() + u) >> 20).clamp(max=0x7E)
        c = torch.where((c == 0) & (x > 0) & (s > 0), torch.ones_like(c), c)
        out += [c.to(torch.uint8), s.view(-1)]
    return out


@pytest.mark.parametrize("n", [1, 300, 256 * 9 + 17, 256 * 40 + 3])
def test_adamw8_codes_are_reproducible(n):
    """The stored bits are those of the documented arithmetic: fp32 operations one by one, the documented random bits. Equal, not near: no
    operation of the step is fused, approximated or dependent on where a lane lies. (first step: the moments are (1 - b1) g, (1 - b2) g^2.)"""
    g = torch.randn(n, generator=gen(n), device=DEV) * torch.exp2(torch.randint(-12, 1, (n,), generator=gen(n + 1), device=DEV).float())
    p = torch.zeros(n, device=DEV)
    st, steps = O.AdamState8.zeros([p]), torch.full((1,), 41, dtype=torch.int32, device=DEV)
    O.adamw8_step([p], [g], st, steps, lr=1.0)
    f = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
    gc = g.cpu()
    m = torch.zeros(n) * f(0.9) + gc * f(1 - 0.9)
    v = torch.zeros(n) * f(0.999) + (gc * gc) * f(1 - 0.999)
    # the IEEE square root: torch's fp32 one on the CPU can be one unit off; rounded to fp32 the root in 64 bits is exact (53 >= 2 * 24 + 2 bits)
    cm, sm, cr, sr = plain8(m, v.double().sqrt().float(), 42)
    assert torch.equal(st.exp_avg_scale[0].cpu(), sm) and torch.equal(st.root_scale[0].cpu(), sr)
    assert torch.equal(st.exp_avg[0].view(torch.uint8).cpu(), cm.view(-1)[:n])
    assert torch.equal(st.root[0].view(torch.uint8).cpu(), cr.view(-1)[:n])


def test_roots_keep_their_expected_value():
    """Without gradients the second moment falls by 0.1 % a step, a 1/100th of the distance between codes. After 200 steps the mean over N elements
    of the stored root has to be 0.999^100 of the start's. A step rounds by a variable of variance f (1 - f) d^2, d = the distance (2^-3 at 1.x
    .. in units of the binade), f <= 0.0005 x / d: over 200 steps and N elements the mean's deviation is at most sqrt(200 * 0.0005 x d / N)."""
    n = 256 * 256
    r = torch.full((n,), 1.5, device=DEV)
    r[::BLOCK] = 448.0                               # every block's scale is 1 at the start and falls as the roots do
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    st, steps = O.AdamState8.zeros([p]), torch.zeros(1, dtype=torch.int32, device=DEV)
    O.write_adam_state8(st, [torch.zeros(n, device=DEV)], [r * r])
    # hold the scale: the first element of each block gets the gradient that keeps its second moment
    g[::BLOCK] = 448.0
    for _ in range(200):
        O.adamw8_step([p], [g], st, steps, lr=0.0)
    got = rows(st.root[0].float()).double() * st.root_scale[0].double().view(-1, 1)
    got = got[:, 1:].mean()
    want = 1.5 * 0.999 ** 100
    sigma = math.sqrt(200 * 0.0005 * 1.5 * 0.125 / n)
    # the root is convex in the second moment's rounding: E[sqrt] of a spread of variance w is below sqrt(E) by w / (8 r^3) of (r^2)'s variance, and
    # the moment is kept in the root: no bias from there. 6 sigma, and fp32's 200 roundings.
    assert abs(float(got) - want) < 6 * sigma + 200 * 8 * U * want
    assert len(torch.unique(st.root[0].view(torch.uint8))) > 2


def test_adamw8_zero_tiny_and_not_finite_blocks():
    n = BLOCK * 6 + 5
    p, g = torch.ones(n, device=DEV), torch.randn(n, generator=gen(1), device=DEV)
    g[:BLOCK] = 0                                    # a block without gradients
    g[BLOCK:2 * BLOCK] *= 1e-30                      # squares that underflow: v = 0, m below the least scale is kept or flushed, never NaN
    g[2 * BLOCK:3 * BLOCK] *= 1e-18
    g[3 * BLOCK + 7] = math.nan
    g[4 * BLOCK + 9] = math.inf
    g[5 * BLOCK:] *= 1e18
    st, steps = O.AdamState8.zeros([p]), torch.zeros(1, dtype=torch.int32, device=DEV)
    O.adamw8_step([p], [g], st, steps, lr=1e-3, weight_decay=0.0)
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[3 * BLOCK + 7] = bad[4 * BLOCK + 9] = True
    assert torch.equal(torch.isfinite(p), ~bad) and bool((p[:BLOCK] == 1).all())
    m, v = [torch.zeros(n, device=DEV)], [torch.zeros(n, device=DEV)]
    O.read_adam_state8(st, m, v)
    fine = torch.ones(n, dtype=torch.bool, device=DEV)
    fine[3 * BLOCK:5 * BLOCK] = False                # the whole block of an element that is not finite reads back as NaN
    assert torch.equal(torch.isfinite(m[0]), fine) and torch.equal(torch.isfinite(v[0]), fine)
    assert not m[0][:BLOCK].any() and not v[0][:BLOCK].any()
    assert bool((st.root[0][5 * BLOCK:].float() > 0).all())


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", [SIZES, SMALL])
def test_state8_write_and_read(shift, sizes):
    x = make(sizes + [0], torch.float32, seed=20, shift=shift)
    st = O.AdamState8.zeros(x["p"])
    O.write_adam_state8(st, x["m"], x["v"])
    for i in range(len(sizes)):
        r = x["v"][i].double().sqrt()
        check8(st, i, x["m"][i].double(), torch.zeros_like(r), r, U * r + 2.0 ** -149, True)
    back = make(sizes + [0], torch.float32, seed=21, shift=shift)
    O.read_adam_state8(st, back["m"], back["v"])
    for i in range(len(sizes)):
        m = (rows(st.exp_avg[i].float()) * st.exp_avg_scale[i].view(-1, 1)).view(-1)[:sizes[i]]
        r = (rows(st.root[i].float()) * st.root_scale[i].view(-1, 1)).view(-1)[:sizes[i]]
        assert torch.equal(back["m"][i], m) and torch.equal(back["v"][i], r * r)
    assert all(guards_intact(v, b, shift) for v, b in back["buf"])
    again = O.AdamState8.zeros(x["p"])               # what was read is written back to the same codes
    O.write_adam_state8(again, back["m"], back["v"])
    for a, b in zip(st.exp_avg + st.root, again.exp_avg + again.root):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_every_code_converts_like_torch():
    """The conversion instructions against torch's e4m3: all 127 magnitudes and the points between them, both signs."""
    c = torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).float()
    mid = (c[1:] + c[:-1]) / 2
    x = torch.cat([c, mid, torch.nextafter(mid, torch.zeros_like(mid)), torch.nextafter(mid, torch.full_like(mid, 500.0))])
    x = torch.cat([x, -x])
    n = x.numel()
    x = torch.nn.functional.pad(x, (0, -n % (BLOCK - 1))).view(-1, BLOCK - 1)
    x = torch.nn.functional.pad(x, (1, 0), value=448.0).view(-1)       # every block's scale is 1
    st = O.AdamState8.zeros([x])
    O.write_adam_state8(st, [x], [torch.zeros_like(x)])
    assert bool((st.exp_avg_scale[0] == 1).all())
    assert torch.equal(st.exp_avg[0].float(), x.to(torch.float8_e4m3fn).float())


# ---- norm and clipping

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", [SIZES, SMALL])
def test_norm_and_clip(dtype, shift, sizes):
    x = make(sizes + [0, 1], dtype, seed=30 + shift, shift=shift)
    g0 = [g.double() for g in x["g"]]
    norm = math.sqrt(sum(float(g.square().sum()) for g in g0))
    assert abs(float(O.grad_norm(x["g"])) - norm) <= 2 * U * norm
    assert abs(float(O.grad_norm(x["g"], torch.tensor(3.0, device=DEV))) - norm / 3) <= 2 * U * norm / 3
    keep = [g.clone() for g in x["g"]]
    version = x["g"][0]._version
    assert abs(float(O.clip_grads_(x["g"], norm * 1.5)) - norm) <= 2 * U * norm
    assert all(torch.equal(a, b) for a, b in zip(x["g"], keep)) and x["g"][0]._version > version
    got = O.clip_grads_(x["g"], 0.75 * norm)
    assert abs(float(got) - norm) <= 2 * U * norm
    f = 0.75 * norm / (norm + 1e-6)
    for g, w in zip(x["g"], g0):
        within(g, w * f, 4 * U * (w * f).abs() + 2.0 ** -149, dtype)
    assert all(guards_intact(v, b, shift) for v, b in x["buf"])


BETWEEN = [4097, 8191, 8192, 300]                    # one launch for the step, several for the norm
TILE = 4096                                          # of clipping alone (the step's: 2048)


@pytest.mark.parametrize("sizes", [BETWEEN, BETWEEN + [8193]])
def test_sizes_around_the_kernels_for_small_tensors(sizes):
    for dtype in (torch.float32, torch.bfloat16):
        for shift in (0, 1):
            test_adamw_step(dtype, shift, 3, sizes)
            test_adamw8_step(dtype, shift, 3, sizes)
            test_norm_and_clip(dtype, shift, sizes)
    test_state8_write_and_read(1, sizes)


@pytest.mark.parametrize("sizes", [[TILE * 1023], [TILE * 1023 + 1], [70000] + [5] * 163, [70000] + [5] * 164, [0, 70000, 0, 0, 3] * 32 + [0, 4097]])
def test_norm_and_clip_of_many_tiles_and_tensors(sizes):
    """Few and many partial sums; one type in the kernel arguments and more tensors than they hold, empty ones in between and at the end.
    (test_norm_and_clip adds two tensors, of 0 and 1 elements: 1024 and 1025 tiles, 166 and 167 tensors.)"""
    for dtype in (torch.float32, torch.float16):
        test_norm_and_clip(dtype, 1, sizes)


@pytest.mark.parametrize("tiles", [1000, 1030])
@pytest.mark.parametrize("bits", [32, 8])
def test_one_norm_over_tensors_of_three_types(tiles, bits):
    """The partial sums of every type, in few workgroups (1000 tiles) and in many: all kernels behind them take the same factor."""
    parts = [make([2048 * k, 77, 1, 5000], dtype, seed=40 + k) for k, dtype in ((tiles - 60, torch.float32), (20, torch.bfloat16), (25, torch.float16))]
    x = {k: [t for part in parts for t in part[k]] for k in "pgmv"}
    kinds = [t.dtype for t in x["p"]]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in x["g"]))
    factor = 0.25 * norm / (norm + 1e-6)
    steps = torch.full((len(kinds),), 4, dtype=torch.int32, device=DEV)
    if bits == 8:
        st = O.AdamState8.zeros(x["p"])
        want = [formula(p, g, m * 0, v * 0, 5, 1e-2, 0.9, 0.999, 1e-8, 0.1, factor) for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"])]
        got = O.adamw8_step(x["p"], x["g"], st, steps, lr=1e-2, weight_decay=0.1, max_norm=0.25 * norm)
    else:
        want = [formula(p, g, m, v, 5, 1e-2, 0.9, 0.999, 1e-8, 0.1, factor) for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"])]
        got = O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=1e-2, weight_decay=0.1, max_norm=0.25 * norm)
    assert abs(float(got) - norm) <= 2 * U * norm
    for p, dtype, (wp, _, _) in zip(x["p"], kinds, want):
        within(p, wp[0], 1.5 * wp[1], dtype)
    clipped = [g.double() * factor for g in x["g"]]
    assert abs(float(O.clip_grads_(x["g"], 0.25 * norm)) - norm) <= 2 * U * norm
    for g, w, dtype in zip(x["g"], clipped, kinds):
        within(g, w, 4 * U * w.abs() + 2.0 ** -149, dtype)


def test_norm_of_extremes():
    n = lambda *v: float(O.grad_norm([torch.tensor(v, device=DEV)]))  # noqa: E731
    assert n(0.0) == 0.0 and n(3e38, 1e30) == pytest.approx(3e38) and n(1e-30, 0.0) == pytest.approx(1e-30, rel=1e-6)
    assert math.isinf(n(1.0, math.inf)) and math.isnan(n(1.0, math.nan)) and math.isinf(n(3e38, 3e38))
    assert float(O.grad_norm([])) == 0.0 and float(O.clip_grads_([], 1.0)) == 0.0
    g = torch.tensor([1.0, math.inf, math.nan], device=DEV)
    O.clip_grads_([g], 1.0)
    assert bool(torch.isnan(g).all())                # as in torch.nn.utils.clip_grad_norm_
    z = torch.zeros(300, device=DEV)
    assert float(O.clip_grads_([z], 0.0)) == 0.0 and not z.any()
    one = torch.ones(4, device=DEV)
    O.clip_grads_([one], 0.0)
    assert not one.any()


def test_clip_grad_norm_like_torch():
    g = gen(33)
    mk = lambda: [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((4, 5, 3), (700,), (33, 3), (5,))]  # noqa: E731
    a, b = mk(), mk()
    for p, q in zip(a[:3], b[:3]):                   # the last one has no gradient
        p.grad = torch.randn(p.shape, generator=g, device=DEV)
        q.grad = p.grad.clone()
    a[2].grad = torch.randn(33, 6, generator=g, device=DEV)[:, ::2]
    b[2].grad = a[2].grad.clone()
    ta = O.clip_grad_norm_(a, 2.0)
    tb = torch.nn.utils.clip_grad_norm_(b, 2.0)
    # torch sums squares in fp32: 900 of them in some order, at most 900 u (half of it in the root)
    assert abs(float(ta) - float(tb)) <= 500 * U * float(tb)
    for p, q in zip(a[:3], b[:3]):
        assert bool(((p.grad - q.grad).abs() <= 510 * U * q.grad.abs()).all())


def test_norm_does_not_depend_on_the_run():
    x = make([1 << 20, 77777, 5], torch.float32, seed=34)
    a = [float(O.grad_norm(x["g"])) for _ in range(5)]
    assert len(set(a)) == 1


# ---- as they are used

def network(seed, dtype=torch.float32):
    torch.manual_seed(seed)
    net = torch.nn.Sequential(torch.nn.Conv3d(2, 8, 3, padding=1), torch.nn.GroupNorm(2, 8), torch.nn.ReLU(), torch.nn.Conv3d(8, 40, 3, padding=1), torch.nn.ReLU(),
                              torch.nn.Flatten(), torch.nn.Linear(40 * 64, 11))
    return net.to(DEV, dtype)


def loss_of(net, seed):
    x = torch.randn(3, 2, 4, 4, 4, generator=gen(seed), device=DEV, dtype=next(net.parameters()).dtype)
    return net(x).float().square().mean()


def clone_moments(opt):
    return {i: {k: v.clone() for k, v in st.items()} for i, st in opt.state_dict()["state"].items()}


def test_optimizer_against_torch():
    """AdamW and torch.optim.AdamW from the same state and gradients: one step differs by the two implementations' roundings, twice `formula`'s bounds."""
    net = network(0)
    ps = list(net.parameters())
    groups = lambda q: [{"params": q[::2], "weight_decay": 0.1}, {"params": q[1::2], "weight_decay": 0.0}]  # noqa: E731
    opt = O.AdamW(groups(ps), lr=2e-3)
    for k in range(4):
        opt.zero_grad()
        loss_of(net, k).backward()
        qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        ref = torch.optim.AdamW(groups(qs), lr=2e-3)
        if k:                                        # (torch's load_state_dict keeps the tensors it is given)
            ref.load_state_dict({**opt.state_dict(), "state": clone_moments(opt)})
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        zeros = torch.zeros(())
        order = [p.detach() for p in ps[::2] + ps[1::2]]
        given = [p.grad.clone() for p in ps[::2] + ps[1::2]]
        old = {i: (s["exp_avg"].clone(), s["exp_avg_sq"].clone()) for i, s in opt.state_dict()["state"].items()}
        want = [formula(p, given[i], *(old.get(i) or (zeros.to(DEV).expand(p.shape),) * 2), k + 1, 2e-3, 0.9, 0.999, 1e-8, 0.1 if i < len(ps[::2]) else 0.0)
                for i, p in enumerate(order)]
        opt.step()
        ref.step()
        theirs = [q.detach() for q in qs[::2] + qs[1::2]]
        for p, q, (wp, wm, wv) in zip(order, theirs, want):
            within(p, *wp)
            assert bool(((p - q).abs().double() <= 2 * wp[1] + 8 * U * wp[0].abs()).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_training_loop_with_scaler_clipping_and_schedule(bits):
    """The operators together, as a user runs them: autocast, GradScaler, AdamW with clipping, a schedule, checkpoint in the middle; an overflow step
    leaves everything alone. The resumed run is the uninterrupted one, bit by bit."""
    def setup():
        net = network(1)
        opt = O.AdamW(net.parameters(), lr=1e-2, state_bits=bits, max_norm=0.5, min_8bit_numel=1000)
        return net, opt, O.LinearWarmupPolyLR(opt, 3, 1e-4, 0.9, 20), torch.amp.GradScaler("cuda", init_scale=2.0 ** 10)

    def train(net, opt, sched, scaler, first, last):
        for k in range(first, last):
            opt.zero_grad()
            with torch.autocast("cuda", dtype=torch.float16):
                loss = loss_of(net, k)
            scaler.scale(loss).backward()
            if k == 2:
                next(net.parameters()).grad.view(-1)[0] = math.inf
            before = [p.detach().clone() for p in net.parameters()]
            scaler.step(opt)
            scaler.update()
            sched.step()
            if k == 2:
                assert all(torch.equal(a, b) for a, b in zip(before, net.parameters())) and scaler.get_scale() == 2.0 ** 9
            else:
                assert not torch.equal(before[0], next(net.parameters())) and math.isfinite(float(opt.grad_norm))

    a = setup()
    train(*a, 0, 5)
    sd, so, ss, sc = ({k: v.clone() for k, v in a[0].state_dict().items()}, a[1].state_dict(), a[2].state_dict(), a[3].state_dict())
    so = {"state": clone_moments(a[1]), "param_groups": so["param_groups"]}
    kinds = {8 if "root" in s else 32 for s in so["state"].values()}
    assert kinds == ({32} if bits == 32 else {8, 32}) and {float(s["step"]) for s in so["state"].values()} == {4.0}
    b = setup()
    b[0].load_state_dict(sd), b[1].load_state_dict(so), b[2].load_state_dict(ss), b[3].load_state_dict(sc)
    grads = []
    for net, opt, sched, scaler in (a, b):           # one more step from gradients that are given (the backward pass has atomics)
        for i, p in enumerate(net.parameters()):
            p.grad = torch.randn(p.shape, generator=gen(50 + i), device=DEV) * scaler.get_scale()
        scaler.scale(torch.zeros((), device=DEV))
        scaler.step(opt)
        scaler.update()
        grads.append([p.detach().clone() for p in net.parameters()] + [t.float() for st in opt.state_dict()["state"].values() for t in st.values()])
    assert all(torch.equal(x, y) for x, y in zip(*grads))


def test_parameters_that_change_their_type_or_share_memory():
    """A module may be cast after its state was made (the moments stay as they are), gradients may lie in another order than their parameters, and two
    parameters on one piece of memory are refused."""
    for strided in (False, True):
        g = gen(60)
        p = torch.nn.Parameter(torch.randn(40, 300, generator=g, device=DEV))
        opt = O.AdamW(p, lr=1e-2, weight_decay=0.0)
        fresh = lambda: torch.randn(300, 40, generator=g, device=DEV).t() if strided else torch.randn(40, 300, generator=g, device=DEV)  # noqa: E731
        p.grad = fresh()
        opt.step()
        st = opt.state_dict()["state"][0]
        m, v = st["exp_avg"].clone(), st["exp_avg_sq"].clone()
        p.grad = None
        p.data = p.data.bfloat16()
        p.grad = fresh().bfloat16()
        wp, wm, wv = formula(p.detach(), p.grad, m, v, 2, 1e-2, 0.9, 0.999, 1e-8, 0.0)
        opt.step()
        within(p.detach(), *wp, torch.bfloat16)
        within(st["exp_avg"], *wm)
        within(st["exp_avg_sq"], *wv)
        p.data = p.data[:20].clone()
        p.grad = None
        p.grad = torch.zeros_like(p)
        with pytest.raises(L.NndetError, match="changed its size"):
            opt.step()
    base = torch.zeros(100, device=DEV)
    ps = [torch.nn.Parameter(base), torch.nn.Parameter(base.view(10, 10))]
    opt = O.AdamW(ps)
    for q in ps:
        q.grad = torch.ones_like(q)
    for _ in range(2):
        with pytest.raises(L.NndetError, match="twice"):
            opt.step()
    assert not base.any()


def test_any_iterable_is_a_list():
    x = make([700, 33], torch.float32, seed=61)
    y = make([700, 33], torch.float32, seed=61)
    steps, steps2 = (torch.zeros(2, dtype=torch.int32, device=DEV) for _ in range(2))
    O.adamw_step(x["p"], x["g"], x["m"], x["v"], steps, lr=0.1)
    O.adamw_step(iter(y["p"]), tuple(y["g"]), dict(enumerate(y["m"])).values(), (t for t in y["v"]), steps2, lr=0.1)
    assert all(torch.equal(a, b) for k in "pmv" for a, b in zip(x[k], y[k])) and torch.equal(steps, steps2)
    assert all(p._version > 0 for p in y["p"])


@pytest.mark.parametrize("have,want", [(32, 8), (8, 32), (8, 8)])
def test_checkpoints_convert(have, want):
    net = network(2)
    a = O.AdamW(net.parameters(), lr=1e-2, state_bits=have, min_8bit_numel=64)
    for k in range(3):
        a.zero_grad()
        loss_of(net, k).backward()
        a.step()
    b = O.AdamW(net.parameters(), state_bits=want, min_8bit_numel=64)
    b.load_state_dict(a.state_dict())
    fa, fb = a.state_dict(bits=32)["state"], b.state_dict(bits=32)["state"]
    for i, p in enumerate(net.parameters()):
        assert ("root" in b.state_dict()["state"][i]) == (want == 8 and p.numel() >= 64)
        assert float(fb[i]["step"]) == 3.0
        for k in ("exp_avg", "exp_avg_sq"):
            x, y = fa[i][k].double().view(-1), fb[i][k].double().view(-1)
            if have == 8 or want == 32 or p.numel() < 64:
                assert bool(((x - y).abs() <= 4 * U * x.abs()).all())
            else:                                    # one rounding to nearest: half a step, 2^-4 of a value, and 2^-10 of the scale (its square) below
                top = rows(x.abs()).amax(1, keepdim=True).expand(-1, BLOCK).reshape(-1)[:x.numel()]
                lim = 2.0 ** -4 * x.abs() + 2.0 ** -10 * top / 448 if k == "exp_avg" else 0.13 * x.abs() + (2.0 ** -9 / 448) ** 2 * top + 2.0 ** -9 / 448 * (x * top).sqrt()
                assert bool(((x - y).abs() <= lim * 1.001).all())
    t = torch.optim.AdamW(net.parameters(), lr=1e-2)
    t.load_state_dict(b.state_dict(bits=32))
    loss_of(net, 9).backward()
    t.step()


def test_checkpoint_of_another_memory_order():
    """8-bit moments belong to consecutive elements: a checkpoint whose parameters lay in channels-last order loads into contiguous ones by value."""
    w = torch.randn(8, 16, 3, 3, 3, generator=gen(70), device=DEV)
    g = torch.randn(8, 16, 3, 3, 3, generator=gen(71), device=DEV) * torch.exp2(torch.arange(16, device=DEV).float() - 8).view(1, 16, 1, 1, 1)
    p, q = torch.nn.Parameter(w.contiguous(memory_format=torch.channels_last_3d)), torch.nn.Parameter(w.clone())
    a, b = O.AdamW([p], state_bits=8, min_8bit_numel=1), O.AdamW([q], state_bits=8, min_8bit_numel=1)
    p.grad = g.contiguous(memory_format=torch.channels_last_3d)
    a.step()
    b.load_state_dict(a.state_dict())
    x, y = a.state_dict(bits=32)["state"][0], b.state_dict(bits=32)["state"][0]
    assert b.state_dict()["state"][0]["exp_avg"].is_contiguous()
    top = g.abs().max() * 0.1
    # one more rounding to nearest: 2^-4 of a value, or 2^-10 of a block's scale (at most the tensor's) below the normal codes
    assert bool(((x["exp_avg"] - y["exp_avg"]).abs() <= 1.001 * torch.maximum(2.0 ** -4 * x["exp_avg"].abs(), 2.0 ** -10 * top / 448)).all())
    rx, ry = x["exp_avg_sq"].double().sqrt(), y["exp_avg_sq"].double().sqrt()
    assert bool(((rx - ry).abs() <= 1.001 * torch.maximum(2.0 ** -4 * rx, 2.0 ** -9 * rx.max() / 448)).all())
    q.grad = g.clone()
    b.step()
    assert bool(torch.isfinite(q).all())


def test_checkpoints_that_do_not_fit():
    p = torch.nn.Parameter(torch.randn(700, device=DEV))
    p.grad = torch.randn_like(p)
    for bits in (8, 32):
        opt = O.AdamW([p], state_bits=bits, min_8bit_numel=1)
        opt.step()
        good = opt.state_dict()
        for k, bad in (("exp_avg", torch.zeros(699, device=DEV)), ("root_scale", torch.zeros(2, device=DEV)), ("exp_avg_scale", torch.zeros(3, device=DEV, dtype=torch.float64)),
                       ("root", torch.zeros(700, device=DEV)), ("exp_avg_sq", torch.zeros(1, device=DEV))):
            st = good["state"][0]
            if k in st:
                with pytest.raises(ValueError, match="do not fit"):
                    O.AdamW([p], state_bits=bits).load_state_dict({**good, "state": {0: {**st, k: bad}}})


def test_optimizer_with_two_rates_clips_by_one_norm():
    net = network(3)
    ps = list(net.parameters())
    opt = O.AdamW([{"params": ps[:3], "lr": 1e-2}, {"params": ps[3:], "lr": 1e-3, "betas": (0.8, 0.9)}], max_norm=0.01, weight_decay=0.0)
    loss_of(net, 0).backward()
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
    want = [formula(p.detach(), p.grad, torch.zeros_like(p), torch.zeros_like(p), 1, 1e-2 if i < 3 else 1e-3, *((0.9, 0.999) if i < 3 else (0.8, 0.9)), 1e-8, 0.0,
                    0.01 / (norm + 1e-6)) for i, p in enumerate(ps)]
    opt.step()
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    for p, w in zip(ps, want):
        within(p.detach(), w[0][0], 1.5 * w[0][1])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    """Two graphs of one optimiser (each with its own workspace), replayed in turn with eager steps and a schedule between: like eager steps."""
    def setup():
        net = network(4)
        lr = torch.tensor(1e-2, device=DEV)
        opt = O.AdamW(net.parameters(), lr=lr, state_bits=bits, max_norm=1.0, min_8bit_numel=256)
        for i, p in enumerate(net.parameters()):
            p.grad = torch.randn(p.shape, generator=gen(i), device=DEV)
        return list(net.parameters()), lr, opt

    def fresh(ps, k):
        for i, p in enumerate(ps):
            p.grad.copy_(torch.randn(p.shape, generator=gen(1000 * k + i), device=DEV))

    ps, lr, opt = setup()
    qs, lr2, ref = setup()
    stream = torch.cuda.Stream()
    bare = O.AdamW([torch.nn.Parameter(torch.zeros(4, device=DEV))])
    bare.param_groups[0]["params"][0].grad = torch.zeros(4, device=DEV)
    torch.cuda.synchronize()
    opt.step(), ref.step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            opt.step()
            with pytest.raises(L.NndetError, match="outside of the capture"):
                bare.step()
        graphs.append(g)
    for k in range(7):
        lr.fill_(1e-2 / (k + 1)), lr2.fill_(1e-2 / (k + 1))
        fresh(ps, k), fresh(qs, k)
        if k == 3:
            opt.step()
        else:
            graphs[k % 2].replay()
        ref.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps, qs)), k
        for a, b in zip(opt.state_dict()["state"].values(), ref.state_dict()["state"].values()):
            assert all(torch.equal(a[x].float(), b[x].float()) for x in a)


@pytest.mark.parametrize("most", [4000, 100000])
def test_captured_clip_and_another_stream(most):
    """Clipping in a graph, replayed with fresh gradients; then the same call on a side stream."""
    x = make([3000, 17, most], torch.float32, seed=40)
    fresh = [torch.randn(g.shape, generator=gen(41 + i), device=DEV) for i, g in enumerate(x["g"])]
    O.clip_grads_(x["g"], 1.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = O.clip_grads_(x["g"], 1.0)
    for k in range(5):
        for a, b in zip(x["g"], fresh):
            a.copy_(b * (k + 1))
        want = [a.clone() for a in x["g"]]
        g.replay()
        torch.cuda.synchronize()
        n = O.clip_grads_(want, 1.0)
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(x["g"], want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(x["g"], fresh):
            a.copy_(b)
        n2 = O.clip_grads_(x["g"], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, fresh):
        a.copy_(b)
    n = O.clip_grads_(want, 1.0)
    assert torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(x["g"], want))


def test_a_tensor_past_32_bit_offsets():
    """2^31 + 1500 bf16 parameters: offsets in elements and bytes past 32 bits. Slices at the start, around 2^31 / 2^32 bytes and at the end."""
    n = (1 << 31) + 1500
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    at = [0, (1 << 29) - 500, (1 << 30) - 500, (1 << 31) - 700, n - 1000]
    for i, a in enumerate(at):
        g[a:a + 1000] = torch.randn(1000, generator=gen(i), device=DEV).bfloat16()
        p[a:a + 1000] = torch.randn(1000, generator=gen(90 + i), device=DEV).bfloat16()
    want = [formula(p[a:a + 1000], g[a:a + 1000], m[a:a + 1000], v[a:a + 1000], 1, 1e-2, 0.9, 0.999, 1e-8, 0.01) for a in at]
    norm = math.sqrt(sum(float(g[a:a + 1000].double().square().sum()) for a in (at[0], at[1], at[2], at[3])) + float(g[at[3] + 1000:].double().square().sum()))
    assert abs(float(O.grad_norm([g])) - norm) <= 2 * U * norm
    st = O.AdamState8.zeros([p])
    q = p.clone()
    O.adamw_step([p], [g], [m], [v], torch.zeros(1, dtype=torch.int32, device=DEV), lr=1e-2)
    O.adamw8_step([q], [g], st, torch.zeros(1, dtype=torch.int32, device=DEV), lr=1e-2)
    for a, (wp, wm, wv) in zip(at, want):
        within(p[a:a + 1000], *wp, torch.bfloat16)
        within(m[a:a + 1000], *wm)
        within(v[a:a + 1000], *wv)
    assert torch.equal(p, q)                         # (a first step: both computed from moments of zero)
    assert int((m != 0).sum()) == int((g != 0).sum())


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_the_networks_training_step(kind):
    """configure_optimizer(optimizer=...) on the detection network: a training step through the HIP modules moves every parameter that has a gradient by
    what the formula says, and the packed weights follow."""
    from nndetection_amd.plans import TRAINER_CFG_V001, get_plan
    from nndetection_amd.ptmodule import build_model, configure_optimizer
    from tests.gpu_util import synth_inputs
    plan = get_plan("tiny")
    torch.manual_seed(0)
    net = build_model(plan).to(DEV)
    opt, sched = configure_optimizer(net, dict(TRAINER_CFG_V001, optimizer=kind, max_norm=12.0, warm_iterations=2, initial_lr=1e-3))
    x, targets = synth_inputs(plan)
    targets = {k: ([t.to(DEV) for t in v] if isinstance(v, list) else v.to(DEV)) for k, v in targets.items()}
    losses = []
    for k in range(3):
        opt.zero_grad()
        loss_dict, _ = net.train_step(images=x.to(DEV), targets=targets, evaluation=False, batch_num=k)
        loss = sum(loss_dict.values())
        loss.backward()
        losses.append(float(loss.detach()))
        if k == 0:
            named = [(p, g["weight_decay"], p.detach().clone(), p.grad.clone()) for g in opt.param_groups for p in g["params"] if p.grad is not None]
            lr = opt.param_groups[0]["lr"]
        opt.step()
        if k == 0:
            norm = math.sqrt(sum(float(g.double().square().sum()) for _, _, _, g in named))
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
            for p, wd, old, g in named:
                wp, _, _ = formula(old, g, torch.zeros_like(old), torch.zeros_like(old), 1, lr, 0.9, 0.999, 1e-8, wd, min(1.0, 12.0 / (norm + 1e-6)))
                within(p.detach(), wp[0], 1.5 * wp[1])
        sched.step()
    assert all(math.isfinite(v) for v in losses) and len(set(losses)) == 3      # the network saw other weights each time
