"""Optimisers of the training step: lean SGD(nesterov), AdamW with moments in 32 or in 8 bits, clipping by the global gradient norm, and
LinearWarmupPolyLR.

SGD: same update rule as `torch.optim.SGD(momentum, nesterov, weight_decay)` as configured by the reference
(nndet/ptmodule/retinaunet/base.py:300-336) and the same per-iteration schedule as `LinearWarmupPolyLR`
(nndet/training/learning_rate.py:26-57,127-184), but issued as a handful of `torch._foreach_*` launches over static
tensor lists: torch.optim's per-step Python bookkeeping cost ~5 ms of GPU idle time per step after backward
(profiles/round1_v2_kernel_stats.txt gap analysis), which is 10 % of the whole step at MI355X speed.

AdamW and clipping: HIP kernels over all tensors of a call at once (csrc/optim.hip). `AdamW` is the optimiser; `adamw_step`, `adamw8_step`,
`grad_norm`, `clip_grads_`, `write_adam_state8` and `read_adam_state8` are the same operators on lists of tensors. They run on torch's
current stream of the tensors' device, never wait for the GPU, and can be captured into a HIP graph.
"""
import array
import ctypes as C
import operator
import os
import struct
from typing import List, NamedTuple, Optional, Sequence, Union

import torch

from . import _lib as L


def _bump_versions(tensors) -> None:
    """`torch._fused_sgd_` writes the parameters WITHOUT incrementing their autograd version counters (measured on torch 2.10, CPU and
    ROCm; the `_foreach_*` ops do increment them). Everything that caches something derived from a parameter keys it on `_version` --
    here the packed / cast convolution weights (arch/conv.py: _packed) -- so the counters are advanced by hand after the launch."""
    setter = getattr(torch._C._autograd, "_unsafe_set_version_counter", None)
    if setter is not None:
        try:
            setter(tuple(tensors), tuple(t._version + 1 for t in tensors))
            return
        except TypeError:                                      # a torch build whose private setter takes (Tensor, int)
            try:
                for t in tensors:
                    setter(t, t._version + 1)
                return
            except TypeError:
                pass
    torch._foreach_add_(list(tensors), 0.0)                    # an in-place no-op that does bump


class SGDNesterov:
    def __init__(self, param_groups: List[dict], lr: float, momentum: float = 0.9, nesterov: bool = True):
        self.param_groups = []
        for g in param_groups:
            params = [p for p in g["params"] if p.requires_grad]
            self.param_groups.append({"params": params, "weight_decay": float(g.get("weight_decay", 0.0)), "lr": lr})
        self.momentum, self.nesterov = momentum, nesterov
        self.defaults = {"lr": lr, "momentum": momentum, "nesterov": nesterov}
        self._buf = {}

    fused = os.environ.get("NNDET_FUSED_SGD", "1") != "0"   # one multi-tensor launch per group (torch._fused_sgd_, the kernel behind torch.optim.SGD(fused=True))

    # Loss scaling without a host synchronisation (fp16 activations, the reference's precision=16): torch.amp.GradScaler.step() hands
    # an optimizer with this flag the scale and the found-inf flag as DEVICE tensors (attributes `grad_scale` / `found_inf`) instead of
    # reading found_inf on the host; the fused kernel divides the gradients by the scale and skips the update when an inf / nan was
    # found. (The stock path -- torch.optim.SGD without fused=True, what the reference configures -- costs one `.item()` per step.)
    _step_supports_amp_scaling = True

    @torch.no_grad()
    def step(self):
        grad_scale, found_inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        for g in self.param_groups:
            ps = [p for p in g["params"] if p.grad is not None]
            if not ps:
                continue
            grads = [p.grad for p in ps]
            wd, lr, mu = g["weight_decay"], g["lr"], self.momentum
            if (self.fused and mu != 0.0 and hasattr(torch, "_fused_sgd_")
                    and all(p.is_cuda and p.dtype == torch.float32 and gr.dtype == torch.float32 for p, gr in zip(ps, grads))):
                # weight decay, momentum, Nesterov and the update in ONE pass over (p, g, buf) instead of 4-5 foreach passes
                new = {id(p) for p in ps if p not in self._buf}
                for first in (True, False):
                    sel = [(p, gr) for p, gr in zip(ps, grads) if (id(p) in new) == first]
                    if not sel:
                        continue
                    if first:
                        for p, gr in sel:
                            self._buf[p] = torch.empty_like(gr)               # filled by the kernel: buf = g (+ wd * p)
                    torch._fused_sgd_([p for p, _ in sel], [gr.contiguous() for _, gr in sel], [self._buf[p] for p, _ in sel],
                                      weight_decay=wd, momentum=mu, lr=lr, dampening=0.0, nesterov=self.nesterov, maximize=False,
                                      is_first_step=first, grad_scale=grad_scale, found_inf=found_inf)
                _bump_versions(ps)
                continue
            if found_inf is not None and bool(found_inf.item()):      # foreach fallback (CPU / NNDET_FUSED_SGD=0): host decision
                return
            if grad_scale is not None:
                grads = torch._foreach_div(grads, float(grad_scale.item()))
            if wd != 0.0:
                grads = torch._foreach_add(grads, ps, alpha=wd)          # g + wd * p (new tensors, p.grad untouched)
            if mu != 0.0:
                new_ids = {id(p) for p in ps if p not in self._buf}
                for p, gr in zip(ps, grads):                              # first step: buf = g (torch.optim.SGD semantics)
                    if id(p) in new_ids:
                        self._buf[p] = gr.clone()
                old = [(p, gr) for p, gr in zip(ps, grads) if id(p) not in new_ids]
                if old:
                    bufs_old = [self._buf[p] for p, _ in old]
                    torch._foreach_mul_(bufs_old, mu)
                    torch._foreach_add_(bufs_old, [gr for _, gr in old])
                bufs = [self._buf[p] for p in ps]
                if self.nesterov:
                    grads = torch._foreach_add(grads, bufs, alpha=mu)
                else:
                    grads = bufs
            torch._foreach_add_(ps, grads, alpha=-lr)

    # ---- checkpointing, laid out like torch.optim.SGD.state_dict(): {"state": {param index: {"momentum_buffer": t}},
    # "param_groups": [{"lr", "momentum", "nesterov", "weight_decay", "params": [indices]}]} (indices run over the groups in order),
    # so a checkpoint written by torch.optim.SGD with the same parameter groups loads here and vice versa.
    def state_dict(self) -> dict:
        state, groups, idx = {}, [], 0
        for g in self.param_groups:
            ids = []
            for p in g["params"]:
                if p in self._buf:
                    state[idx] = {"momentum_buffer": self._buf[p]}
                ids.append(idx); idx += 1
            groups.append({"lr": g["lr"], "momentum": self.momentum, "dampening": 0, "nesterov": self.nesterov,
                           "weight_decay": g["weight_decay"], "params": ids})
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, sd: dict) -> None:
        groups = sd["param_groups"]
        if len(groups) != len(self.param_groups) or any(len(a["params"]) != len(b["params"]) for a, b in zip(groups, self.param_groups)):
            raise ValueError("loaded state dict has different parameter groups")
        flat = [p for g in self.param_groups for p in g["params"]]
        self._buf = {}
        for k, st in sd["state"].items():
            buf = st.get("momentum_buffer")
            if buf is not None:
                p = flat[int(k)]
                self._buf[p] = buf.detach().to(device=p.device, dtype=p.dtype).clone()
        for g, src in zip(self.param_groups, groups):
            g["lr"], g["weight_decay"] = float(src["lr"]), float(src["weight_decay"])
        if groups:
            self.momentum, self.nesterov = float(groups[0]["momentum"]), bool(groups[0]["nesterov"])

    def zero_grad(self, set_to_none: bool = True):
        for g in self.param_groups:
            for p in g["params"]:
                if set_to_none:
                    p.grad = None
                elif p.grad is not None:
                    p.grad.zero_()


# ---- operators over lists of tensors ------------------------------------------------------------------------------------------------

STATE8_BLOCK = 256                                   # consecutive elements of a tensor that share one scale of the 8-bit moments
_F8 = torch.float8_e4m3fn


class AdamState8(NamedTuple):
    """AdamW moments in 8 bits, one entry a tensor in every list. exp_avg / root: float8_e4m3fn codes in the parameter's shape and memory
    order, of the first moment and of the SQUARE ROOT of the second; exp_avg_scale / root_scale: fp32, one value for each STATE8_BLOCK
    consecutive elements (in memory order). A moment is code * scale."""
    exp_avg: Sequence[torch.Tensor]
    exp_avg_scale: Sequence[torch.Tensor]
    root: Sequence[torch.Tensor]
    root_scale: Sequence[torch.Tensor]

    @staticmethod
    def zeros(params: Sequence[torch.Tensor]) -> "AdamState8":
        """The state before the first step of `params`."""
        codes = lambda: [torch.zeros_like(p, dtype=torch.uint8).view(_F8) for p in params]  # noqa: E731
        scales = lambda: [torch.zeros((-(-p.numel() // STATE8_BLOCK),), dtype=torch.float32, device=p.device) for p in params]  # noqa: E731
        return AdamState8(codes(), scales(), codes(), scales())


def _dense(t: torch.Tensor) -> bool:
    """Do the elements fill one piece of memory, in any order of the dimensions, each place once, as they are (no negation that is still to come)?"""
    if t.is_neg():
        return False
    if t.is_contiguous():
        return True
    size = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != size:
            return False
        size *= n
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Have two dense tensors of one shape the same memory order?"""
    return all(x == y or n == 1 for x, y, n in zip(a.stride(), b.stride(), a.shape)) or a.numel() == 0


def _refuse(what: str):
    raise L.NndetError(what)


def _check_list(name: str, ts, dtype, device, like=None) -> None:
    """Tensors of one type on one GPU, dense; `like`: and of the same sizes and memory order, one for one."""
    for i, t in enumerate(ts):
        if t.device != device:
            _refuse(f"{name}[{i}] is on {t.device}, not on {device}: the tensors of a call are on one GPU")
        if dtype is not None and t.dtype != dtype:
            _refuse(f"{name}[{i}] is {t.dtype}, not {dtype}")
        if like is not None:
            p = like[i]
            if t.shape != p.shape:
                _refuse(f"{name}[{i}] has shape {tuple(t.shape)}, the parameter {tuple(p.shape)}")
            if not (_dense(t) and (t.is_contiguous() and p.is_contiguous() or _same_order(t, p))):
                _refuse(f"{name}[{i}] has strides {t.stride()}, the parameter {p.stride()}: moments lie in the parameter's memory order")
        elif not _dense(t):
            _refuse(f"{name}[{i}] with strides {t.stride()} is not dense in memory")


def _check_lengths(n: int, **lists) -> None:
    for name, ts in lists.items():
        if len(ts) != n:
            _refuse(f"{len(ts)} {name} for {n} tensors")


def _check_distinct(name: str, ts) -> None:
    ptrs = [t.data_ptr() for t in ts if t.numel()]
    if len(set(ptrs)) != len(ptrs):
        _refuse(f"the same tensor twice in {name}: its updates would race")


def _check_read(grads, *written) -> None:
    """No gradient is memory that the call writes for ANOTHER tensor (its own is read before it is written)."""
    at = {t.data_ptr(): i for ts in written for i, t in enumerate(ts) if t.numel()}
    for i, g in enumerate(grads):
        if at.get(g.data_ptr(), i) != i:
            _refuse(f"the gradient of tensor {i} is memory that the call writes for tensor {at[g.data_ptr()]}")


def _scalar(name: str, t, device) -> Optional[int]:
    """Address of a one-element fp32 tensor on `device`, None for None."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.numel() != 1 or t.device != device or t.is_neg():
        _refuse(f"{name} is one fp32 value on {device}")
    return t.data_ptr()


_KIND = {torch.float32: L.F32 << 32, torch.bfloat16: L.BF16 << 32, torch.float16: L.F16 << 32}


def _kinds(ts) -> list:
    try:
        return [_KIND[t.dtype] for t in ts]
    except KeyError as e:
        raise L.NndetError(f"unsupported type {e.args[0]}; use float32, bfloat16 or float16")


def _double_bits(x: float) -> int:
    return struct.unpack("q", struct.pack("d", x))[0]


def _words(n, p, g, m, v, ms, rs, numel, wd, tail) -> bytes:
    """The call's tensors as NndetOptTensor structs (nine 64-bit words each). p .. rs: lists of addresses or None, wd: the bits of doubles or
    None, tail: slot | type << 32 | bits of the moments << 48."""
    zero = [0] * n
    rows = zip(p or zero, g or zero, m or zero, v or zero, ms or zero, rs or zero, numel, wd or zero, tail)
    return array.array("q", [w for row in rows for w in row]).tobytes()


def _run(device, what: str, words, n: int, *args) -> bool:
    """Call `what`(tensors, n, *args, workspace, bytes, stream) on the device's current stream, with a workspace of this call. True if that is being captured."""
    if device.type != "cuda":
        _refuse(f"tensors on {device}: nndetection_amd kernels need tensors on the GPU (no CPU path)")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _run(device, what, words, n, *args)
    nbytes = L.load().nndet_opt_workspace_bytes(n)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=device)
    L.call(what, words, n, *args, ws.data_ptr(), nbytes, L.stream())
    return torch.cuda.is_current_stream_capturing()


def _ptrs(ts) -> list:
    return [t.data_ptr() for t in ts]


def _written(*lists) -> None:
    """The kernels write through raw pointers: advance the version counters as torch's in-place operators do."""
    written = L.host_lists().written
    for ts in lists:
        written(ts, None)


def _pack(device, params, grads, m, v, ms, rs, wd, bits: int, both: bool = False):
    """(structs, number of tensors) of the ordinary call -- everything right, dense, in one memory order and on `device` -- else None, and the checks here
    find out what it is. (92 tensors: 12 us instead of 200.)"""
    return L.host_lists().pack(params, grads, m, v, ms, rs, wd, bits, device.index, both) if device.type == "cuda" else None


def _grads_like(params, grads) -> list:
    """Gradients in the parameters' memory order (a copy where they are not)."""
    out = []
    for i, (p, g) in enumerate(zip(params, grads)):
        if g.layout != torch.strided or g.shape != p.shape:
            _refuse(f"grads[{i}] is {'sparse' if g.layout != torch.strided else 'of shape %s' % (tuple(g.shape),)}, the parameter is dense {tuple(p.shape)}")
        if g.dtype != p.dtype or g.device != p.device:
            _refuse(f"grads[{i}] is {g.dtype} on {g.device}, the parameter {p.dtype} on {p.device}")
        if not (_dense(g) and (g.is_contiguous() and p.is_contiguous() or _same_order(g, p))):
            g = torch.empty_like(p).copy_(g.detach())
        out.append(g)
    return out


Rate = Union[float, torch.Tensor]


def _hyper(lr, betas, eps, max_norm, total_norm, grad_scale, found_inf, steps, device):
    """The scalars of a step as the library takes them, checked, and the norm's tensor (None without clipping)."""
    b1, b2 = float(betas[0]), float(betas[1])
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and (eps == 0.0 or eps >= 2.0 ** -126)):
        _refuse(f"betas {betas} in [0, 1) and an eps {eps} that is 0 or a normal fp32 number are wanted")
    if max_norm is not None and not max_norm >= 0.0:
        _refuse(f"max_norm {max_norm} >= 0 is wanted")
    if total_norm is not None and max_norm is None:
        _refuse("total_norm without max_norm")
    norm = total_norm
    if max_norm is not None and norm is None:
        norm = torch.empty((), dtype=torch.float32, device=device)
    rate = 0.0
    if not isinstance(lr, torch.Tensor):
        lr, rate = None, float(lr)
    elif lr.device.type == "cpu" and device.type != "cpu":
        lr, rate = None, float(lr)
    a = L.NndetAdamw(rate, b1, b2, float(eps), -1.0 if max_norm is None else float(max_norm), _scalar("lr", lr, device),
                     _scalar("grad_scale", grad_scale, device), _scalar("found_inf", found_inf, device), _scalar("total_norm", norm, device),
                     int(total_norm is not None), steps.data_ptr())
    return a, norm


def _listed(*args):
    """Each argument as a list or tuple (None stays None); a class derived from list becomes one."""
    return [x if x is None or type(x) is list or isinstance(x, tuple) else list(x) for x in args]


def _adamw_call(params, grads, m, v, ms, rs, bits, steps, lr, betas, eps, weight_decay, max_norm, total_norm, grad_scale, found_inf):
    params, grads, m, v, ms, rs = _listed(params, grads, m, v, ms, rs)
    n = len(params)
    if bits == 8:
        _check_lengths(n, exp_avg_scale=ms, root_scale=rs)
    _check_lengths(n, grads=grads, exp_avgs=m, exp_avg_sqs=v)
    if not isinstance(steps, torch.Tensor) or steps.dtype != torch.int32 or steps.dim() != 1 or not steps.is_contiguous() or steps.numel() < n:
        _refuse(f"steps is one int32 count a tensor ({n}), contiguous")
    a, norm = _hyper(lr, betas, eps, max_norm, total_norm, grad_scale, found_inf, steps, steps.device)
    packed = _pack(steps.device, params, grads, m, v, ms, rs, weight_decay, bits)
    if packed is not None:
        if _run(steps.device, "nndet_adamw_step", *packed, C.byref(a)):
            L.note_graph_write([p for p, g in zip(params, grads) if g is not None])
        L.host_lists().written(params, grads)
        return norm
    wd = weight_decay if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
    _check_lengths(n, weight_decay=wd)
    slots = range(n)
    if any(g is None for g in grads):                # these tensors and their counts stay as they are
        slots = [i for i, g in enumerate(grads) if g is not None]
        pick = lambda ts: None if ts is None else [ts[i] for i in slots]  # noqa: E731
        params, grads, m, v, ms, rs, wd = (pick(x) for x in (params, grads, m, v, ms, rs, wd))
        n = len(params)
    device = steps.device
    _check_list("params", params, None, device)
    grads = _grads_like(params, grads)
    kinds = _kinds(params)
    for name, ts in (("exp_avgs", m), ("exp_avg_sqs", v)):
        _check_list(name, ts, torch.float32 if bits == 32 else _F8, device, params)
    numel = [p.numel() for p in params]
    if bits == 8:
        for name, ts in (("exp_avg_scale", ms), ("root_scale", rs)):
            _check_scales(name, ts, numel, device)
    _check_distinct("params and moments", [*params, *m, *v, *(ms or ()), *(rs or ())])
    _check_read(grads, params, m, v)
    bits_of = {w: _double_bits(float(w)) for w in set(wd)}
    words = _words(n, _ptrs(params), _ptrs(grads), _ptrs(m), _ptrs(v), ms and _ptrs(ms), rs and _ptrs(rs), numel, [bits_of[w] for w in wd],
                   [s | k | (bits << 48) for s, k in zip(slots, kinds)])
    if _run(device, "nndet_adamw_step", words, n, C.byref(a)):
        L.note_graph_write(params)
    _written(params)
    return norm


def _check_scales(name: str, ts, numel, device) -> None:
    for i, (t, n) in enumerate(zip(ts, numel)):
        if t.dtype != torch.float32 or t.device != device or t.numel() != -(-n // STATE8_BLOCK) or not t.is_contiguous() or t.is_neg():
            _refuse(f"{name}[{i}] is one fp32 value on {device} for each {STATE8_BLOCK} elements of the tensor ({-(-n // STATE8_BLOCK)}), contiguous")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps: torch.Tensor, *, lr: Rate, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay=0.01, max_norm: Optional[float] = None, total_norm: Optional[torch.Tensor] = None,
               grad_scale: Optional[torch.Tensor] = None, found_inf: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """One AdamW step of many tensors in place (torch.optim.AdamW's formula):

        t = steps + 1;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    params / grads: fp32, bf16 or fp16 tensors (any mixture) on one GPU, dense in memory; a gradient in another memory order is copied
    first, a gradient None leaves its tensor, moments and count as they are. exp_avgs / exp_avg_sqs: fp32, in the parameters' memory order.
    steps: int32 counts on the GPU, one a tensor. No two of the tensors may overlap. lr: a number, or one fp32 value on the GPU (a captured
    step follows a schedule through it). weight_decay: a number, or one a tensor. The step is computed in fp32; a 16-bit parameter is rounded
    once, to nearest, so a change below half its unit is lost, as it is in torch.
    max_norm: the gradients are multiplied by min(1, max_norm / (norm + 1e-6)) on the way (they are not written), where norm is `total_norm`
    or else the 2-norm over all gradients of the call; the norm is returned, on the GPU. A norm that is not finite gives what it gives in
    torch's clipping: NaN. grad_scale: the gradients carry this loss scale and are divided by it, before the norm. found_inf: where it is
    not 0 nothing is changed (torch.amp.GradScaler hands both over)."""
    return _adamw_call(params, grads, exp_avgs, exp_avg_sqs, None, None, 32, steps, lr, betas, eps, weight_decay, max_norm, total_norm,
                       grad_scale, found_inf)


def adamw8_step(params, grads, state: AdamState8, steps: torch.Tensor, *, lr: Rate, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01,
                max_norm: Optional[float] = None, total_norm: Optional[torch.Tensor] = None, grad_scale: Optional[torch.Tensor] = None,
                found_inf: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """`adamw_step` with the moments in 8 bits: 2.03 bytes an element instead of 8. The step itself is computed in fp32 from the moments as
    they are stored; the new ones are then rounded, the first to the nearest code, the root of the second up or down with the probability
    that keeps the root's expected value (by bits that follow from the element's index and its step count: the same step gives the same state).
    The expected value of its square is then larger by the variance of the rounding, and the recursion adds that up: with gradients of a fixed
    normal distribution the second moment settles 5 - 6 % too large (2 - 5 % for b2 <= 0.99), its root 1.3 %; state_dict(bits=32) and `read_adam_state8` pass it on.
    A gradient that is not finite makes the moments of its whole block NaN; `found_inf` keeps it out."""
    m, ms, v, rs = state
    return _adamw_call(params, grads, m, v, ms, rs, 8, steps, lr, betas, eps, weight_decay, max_norm, total_norm, grad_scale, found_inf)


def _clip_call(grads, max_norm: float, grad_scale) -> torch.Tensor:
    n = len(grads)
    device = grads[0].device if n else torch.device("cuda", torch.cuda.current_device())
    packed = _pack(device, None, grads, None, None, None, None, 0.0, 0, max_norm >= 0.0)
    if packed is not None:
        norm = torch.empty((), dtype=torch.float32, device=device)
        _run(device, "nndet_grad_clip", *packed, max_norm, _scalar("grad_scale", grad_scale, device), norm.data_ptr())
        if max_norm >= 0.0:
            _written(grads)
        return norm
    for i, g in enumerate(grads):
        if g.layout != torch.strided:
            _refuse(f"grads[{i}] is sparse")
    kinds = _kinds(grads)
    flat = [g if _dense(g) else g.resolve_neg().contiguous() for g in grads]
    _check_list("grads", flat, None, device)
    if max_norm >= 0.0:
        _check_distinct("grads", grads)
        for i, (g, f) in enumerate(zip(grads, flat)):
            if f is not g and any(st == 0 and k > 1 for st, k in zip(g.stride(), g.shape)):
                _refuse(f"grads[{i}] is a broadcast view: several elements share a place and cannot be scaled in place")
    norm = torch.empty((), dtype=torch.float32, device=device)
    words = _words(n, None, _ptrs(flat), None, None, None, None, [g.numel() for g in flat], None, [k | (32 << 48) for k in kinds])
    _run(device, "nndet_grad_clip", words, n, max_norm, _scalar("grad_scale", grad_scale, device), norm.data_ptr())
    if max_norm >= 0.0:
        _written(flat)
        with torch.no_grad():
            for g, f in zip(grads, flat):
                if f is not g:
                    g.copy_(f)
    return norm


def grad_norm(grads, grad_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """2-norm over all `grads` (fp32, bf16 or fp16 on one GPU; squares are summed in fp64) as one fp32 value on the GPU; divided by
    `grad_scale`, one fp32 value there, if they carry a loss scale."""
    return _clip_call([g for g in grads if g is not None], -1.0, grad_scale)


def clip_grads_(grads, max_norm: float) -> torch.Tensor:
    """Multiply `grads` in place by min(1, max_norm / (norm + 1e-6)), norm = their global 2-norm, which is returned (on the GPU, as it was
    before). Nothing is written where the factor is 1."""
    if not max_norm >= 0.0:
        _refuse(f"max_norm {max_norm} >= 0 is wanted")
    return _clip_call([g for g in grads if g is not None], float(max_norm), None)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """`clip_grads_` on the gradients of `parameters` (torch.nn.utils.clip_grad_norm_ for the 2-norm)."""
    if float(norm_type) != 2.0:
        _refuse(f"norm_type {norm_type}: the 2-norm alone is supported")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads_([p.grad for p in parameters], max_norm)


def _state8_call(state: AdamState8, exp_avgs, exp_avg_sqs, write: int) -> None:
    exp_avgs, exp_avg_sqs, *state = _listed(exp_avgs, exp_avg_sqs, *state)
    state = AdamState8(*state)
    n = len(exp_avgs)
    _check_lengths(n, exp_avg_sqs=exp_avg_sqs, exp_avg=state.exp_avg, exp_avg_scale=state.exp_avg_scale, root=state.root, root_scale=state.root_scale)
    if n == 0:
        return
    device = exp_avgs[0].device
    out = state if write else (exp_avgs, exp_avg_sqs)
    packed = _pack(device, exp_avgs, exp_avg_sqs, state.exp_avg, state.root, state.exp_avg_scale, state.root_scale, 0.0, 8, True)
    if packed is not None and exp_avgs[0].dtype == torch.float32:
        _run(device, "nndet_adam_state8", *packed, write)
        return _written(*out)
    _check_list("exp_avgs", exp_avgs, torch.float32, device)
    _check_list("exp_avg_sqs", exp_avg_sqs, torch.float32, device, exp_avgs)
    _check_list("exp_avg", state.exp_avg, _F8, device, exp_avgs)
    _check_list("root", state.root, _F8, device, exp_avgs)
    numel = [t.numel() for t in exp_avgs]
    _check_scales("exp_avg_scale", state.exp_avg_scale, numel, device)
    _check_scales("root_scale", state.root_scale, numel, device)
    _check_distinct("what is written", [t for ts in out for t in ts])
    words = _words(n, _ptrs(exp_avgs), _ptrs(exp_avg_sqs), _ptrs(state.exp_avg), _ptrs(state.root), _ptrs(state.exp_avg_scale), _ptrs(state.root_scale),
                   numel, None, [(L.F32 << 32) | (8 << 48)] * n)
    _run(device, "nndet_adam_state8", words, n, write)
    _written(*out)


def write_adam_state8(state: AdamState8, exp_avgs, exp_avg_sqs) -> None:
    """Round fp32 moments into `state`, in place: the first moments and the roots of the second to the nearest code (a root that is not 0
    to a code that is not 0)."""
    _state8_call(state, exp_avgs, exp_avg_sqs, 1)


def read_adam_state8(state: AdamState8, exp_avgs, exp_avg_sqs) -> None:
    """The moments that `state` stands for into fp32 tensors, in place."""
    _state8_call(state, exp_avgs, exp_avg_sqs, 0)


def _check_group(wd, betas, eps) -> None:
    b1, b2 = betas
    if not (wd >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and (eps == 0.0 or eps >= 2.0 ** -126)):
        _refuse(f"weight_decay {wd} >= 0, betas {(b1, b2)} in [0, 1) and an eps {eps} that is 0 or a normal fp32 number are wanted")


class AdamW:
    """AdamW on the operators above, with the interface of `SGDNesterov`: one call of the library a step for all parameters that share
    (lr, betas, eps), whatever their weight decays and types.

    param_groups: dicts with "params" and optionally "lr", "betas", "eps", "weight_decay"; or the parameters themselves.
    state_bits: 32, or 8 (2 bytes an element for both moments instead of 8); a parameter of fewer than `min_8bit_numel` elements keeps 32
    bits: it would not save anything, and norms and biases have few elements that share a block's scale.
    max_norm: clip by the global gradient norm within the step (the gradients themselves are not written); `grad_norm` holds the norm of
    the last step, on the GPU (None: no parameter had a gradient).
    lr: a number, or one fp32 value on the GPU, which a captured step reads. A step can be captured once every parameter has a state, i.e.
    after a first step outside of the capture. What this package keeps of the parameters (packed weights) follows the replays; what other code keys on
    a parameter's version counter does not see them."""

    _step_supports_amp_scaling = True                # torch.amp.GradScaler hands grad_scale / found_inf over as device tensors

    def __init__(self, param_groups, lr: Rate = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 min_8bit_numel: int = 4096, max_norm: Optional[float] = None):
        if state_bits not in (32, 8):
            _refuse(f"state_bits {state_bits}: 32 or 8")
        if max_norm is not None and not max_norm >= 0.0:
            _refuse(f"max_norm {max_norm} >= 0 is wanted")
        groups = [param_groups] if isinstance(param_groups, torch.Tensor) else list(param_groups)
        if groups and not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        for g in [{"weight_decay": weight_decay, "betas": betas, "eps": eps}, *groups]:
            _check_group(g.get("weight_decay", 0.0), g.get("betas", betas), g.get("eps", eps))
        self.defaults = {"lr": float(lr), "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay}
        self.param_groups = []
        for g in groups:
            more = set(g) - {"params", "lr", "betas", "eps", "weight_decay"}
            if more:
                _refuse(f"unknown entries {sorted(more)} of a parameter group")
            ps = [g["params"]] if isinstance(g["params"], torch.Tensor) else list(g["params"])
            self.param_groups.append({"params": [p for p in ps if p.requires_grad], "lr": g.get("lr", lr), "betas": tuple(g.get("betas", betas)),
                                      "eps": g.get("eps", eps), "weight_decay": float(g.get("weight_decay", weight_decay))})
        flat = [p for g in self.param_groups for p in g["params"]]
        if len(set(map(id, flat))) != len(flat):
            _refuse("a parameter appears twice")
        _kinds(flat)
        self.state_bits, self.min_8bit_numel, self.max_norm = state_bits, int(min_8bit_numel), max_norm
        self.grad_norm: Optional[torch.Tensor] = None
        self._slot = {p: i for i, p in enumerate(flat)}
        self._state = {}                             # parameter -> {name: tensor}
        self._steps = {}                             # device -> int32 counts, one for every parameter
        self._flat = flat                            # in the order of the slots, and the state's tensors in that order (None: no state yet)
        self._lists = tuple([None] * len(flat) for _ in range(4))

    def _bits(self, p) -> int:
        return 8 if self.state_bits == 8 and p.numel() >= self.min_8bit_numel else 32

    def _counts(self, device) -> torch.Tensor:
        if device not in self._steps:
            self._steps[device] = torch.zeros((len(self._slot),), dtype=torch.int32, device=device)
        return self._steps[device]

    def _init_state(self, p) -> None:
        if not _dense(p):
            _refuse(f"a parameter with strides {p.stride()} is not dense in memory")
        if p.device.type != "cuda":
            _refuse(f"a parameter on {p.device}: nndetection_amd kernels need tensors on the GPU (no CPU path)")
        if torch.cuda.is_current_stream_capturing():
            _refuse("a parameter has no state yet: take a step outside of the capture first")
        if self._bits(p) == 8:
            self._set_state(p, dict(zip(AdamState8._fields, (x[0] for x in AdamState8.zeros([p])))))
        else:
            self._set_state(p, {"exp_avg": torch.zeros_like(p, dtype=torch.float32), "exp_avg_sq": torch.zeros_like(p, dtype=torch.float32)})

    def _set_state(self, p, st: dict) -> None:
        self._state[p] = st
        for ts, k in zip(self._lists, ("exp_avg", "root" if "root" in st else "exp_avg_sq", "exp_avg_scale", "root_scale")):
            ts[self._slot[p]] = st.get(k)

    @staticmethod
    def _key(g) -> tuple:
        """What the parameters of one call share."""
        return (id(g["lr"]) if isinstance(g["lr"], torch.Tensor) else g["lr"], *g["betas"], g["eps"])

    def _packed_step(self, device, counts, words, n: int, scale, found) -> None:
        """The step of the `n` tensors in `words` (those of self._flat with a gradient, in order): one call, or one for each key."""
        on = lambda t: None if t is None else t.to(device)  # noqa: E731
        scale, found, total = on(scale), on(found), None
        ps = self._flat if n == len(self._flat) else [p for p in self._flat if p.grad is not None]
        calls = {self._key(g): (g, []) for g in self.param_groups}
        if len(calls) == 1:
            calls = [(g, words, n, ps) for g, _ in calls.values()]
        else:
            i = 0
            for g in self.param_groups:
                of_key = calls[self._key(g)][1]
                for p in g["params"]:
                    if p.grad is not None:
                        of_key.append(i)
                        i += 1
            size = C.sizeof(L.NndetOptTensor)
            calls = [(g, b"".join([words[size * i:size * (i + 1)] for i in own]), len(own), [ps[i] for i in own]) for g, own in calls.values() if own]
            if self.max_norm is not None and len(calls) > 1:     # a norm over all of them first
                total = grad_norm([p.grad for p in ps], scale)
        for g, words, n, ps in calls:
            a, self.grad_norm = _hyper(g["lr"], g["betas"], g["eps"], self.max_norm, total, scale, found, counts, device)
            if _run(device, "nndet_adamw_step", words, n, C.byref(a)):
                L.note_graph_write(ps)
            _written(ps)

    @torch.no_grad()
    def step(self) -> None:
        scale, found = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        self.grad_norm = None
        if len(self._steps) == 1:                    # the ordinary case; None if a state is missing or anything is out of the ordinary
            (device, counts), = self._steps.items()
            flat, wds = self._in_order(), []
            for g in self.param_groups:
                wds += [g["weight_decay"]] * len(g["params"])
            # (a parameter may have been moved to another group, or left out, since the lists were made)
            as_made = len(flat) == len(self._flat) and all(map(operator.is_, flat, self._flat))
            packed = _pack(device, flat, None, *self._lists, wds, 0) if as_made else None
            if packed is not None:
                if packed[1]:
                    self._packed_step(device, counts, *packed, scale, found)
                return
        calls = {}
        for g in self.param_groups:
            wd = _double_bits(float(g["weight_decay"]))
            key = self._key(g)
            for p in g["params"]:
                gr = p.grad
                if gr is None:
                    continue
                if p not in self._state:
                    self._init_state(p)
                slot = self._slot[p]
                m, v, ms, rs = (ts[slot] for ts in self._lists)
                device = m.device
                if p.device != device or p.shape != m.shape or p.is_neg() or (p.stride() != m.stride() and not (_dense(p) and _same_order(p, m))):
                    _refuse(f"a parameter of shape {tuple(p.shape)} on {p.device} was moved or changed its size after its state was made")
                # (its type may have changed: the moments are fp32 or 8 bits whatever it is)
                tail = slot | _kinds([p])[0] | ((32 if ms is None else 8) << 48)
                gr = _grads_like([p], [gr])[0]
                c = calls.get((device, key))
                if c is None:
                    c = calls[(device, key)] = ([], [], [], g)
                c[0].extend((p.data_ptr(), gr.data_ptr(), m.data_ptr(), v.data_ptr(), *((0, 0) if ms is None else (ms.data_ptr(), rs.data_ptr())), p.numel(), wd, tail))
                c[1].append(p)
                c[2].append(gr)
        if not calls:
            return
        on = lambda t, device: None if t is None else t.to(device)  # noqa: E731
        total = None
        if self.max_norm is not None and len(calls) > 1:     # a norm over all of them first
            per = {}
            for (device, _), c in calls.items():
                per.setdefault(device, []).extend(c[2])
            norms = [grad_norm(gs, on(scale, device)) for device, gs in per.items()]
            total = norms[0] if len(norms) == 1 else torch.stack([x.to(norms[0].device, torch.float64) for x in norms]).square().sum().sqrt().float()
        ps, gs = ([t for c in calls.values() for t in c[i]] for i in (1, 2))
        _check_distinct("the parameters", ps)
        _check_read(gs, ps)
        for (device, _), (words, ps, _, g) in calls.items():
            counts = self._counts(device)
            a, self.grad_norm = _hyper(g["lr"], g["betas"], g["eps"], self.max_norm, on(total, device), on(scale, device), on(found, device),
                                       counts, device)
            if _run(device, "nndet_adamw_step", array.array("q", words).tobytes(), len(ps), C.byref(a)):
                L.note_graph_write(ps)
            _written(ps)

    # ---- checkpointing, laid out like torch.optim.AdamW.state_dict(). Parameters with 8-bit moments hold those of `AdamState8` in place of
    # "exp_avg_sq" (resuming from them is exact); bits=32 writes them as fp32 moments, which torch.optim.AdamW loads. load_state_dict takes
    # either kind, its own or torch's, whatever state_bits is here.
    def state_dict(self, bits: Optional[int] = None) -> dict:
        if bits not in (None, 32):
            _refuse(f"state_dict(bits={bits}): 32, or None for the moments as they are")
        state, groups, idx = {}, [], 0
        for g in self.param_groups:
            ids = []
            for p in g["params"]:
                if p in self._state:
                    st = dict(self._state[p])
                    if bits == 32 and "root" in st:
                        full = [torch.empty_like(st["exp_avg"], dtype=torch.float32) for _ in range(2)]
                        read_adam_state8(AdamState8(*([st[k]] for k in AdamState8._fields)), [full[0]], [full[1]])
                        st = dict(zip(("exp_avg", "exp_avg_sq"), full))
                    state[idx] = {"step": self._counts(st["exp_avg"].device)[self._slot[p]].float(), **st}
                ids.append(idx); idx += 1
            groups.append({**{k: v for k, v in g.items() if k != "params"}, "amsgrad": False, "maximize": False, "foreach": None, "capturable": False,
                           "differentiable": False, "fused": None, "decoupled_weight_decay": True, "params": ids})
        return {"state": state, "param_groups": groups}

    def _in_order(self) -> list:
        """The parameters of the groups as they are now: what the numbers in a checkpoint count."""
        ps = []
        for g in self.param_groups:
            ps += g["params"]
        return ps

    def _check_loaded(self, sd: dict) -> None:
        """Everything that load_state_dict wants of a checkpoint, before it touches the optimiser."""
        groups, flat = sd["param_groups"], self._in_order()
        if len(groups) != len(self.param_groups) or any(len(a["params"]) != len(b["params"]) for a, b in zip(groups, self.param_groups)):
            raise ValueError("loaded state dict has different parameter groups")
        if any(g.get("amsgrad") or g.get("maximize") for g in groups):
            raise ValueError("amsgrad and maximize are not supported")
        for i, g in enumerate(groups):
            missing = [k for k in ("lr", "betas", "eps", "weight_decay") if k not in g]
            if missing:
                raise ValueError(f"loaded parameter group {i} has no {', '.join(missing)}")
            float(g["lr"])
            _check_group(float(g["weight_decay"]), g["betas"], float(g["eps"]))
        for k, st in sd["state"].items():
            if not 0 <= int(k) < len(flat):
                raise ValueError(f"loaded state of parameter {k}: there are {len(flat)}")
            p = flat[int(k)]
            names = AdamState8._fields if "root" in st else ("exp_avg", "exp_avg_sq")
            missing = [c for c in ("step", *names) if c not in st]
            if missing:
                raise ValueError(f"loaded state of parameter {k} has no {', '.join(missing)}")
            if not 0 <= float(st["step"]) < 2 ** 31:
                raise ValueError(f"loaded step {st['step']} of parameter {k}")
            blocks = (-(-p.numel() // STATE8_BLOCK),)
            for c in names:
                scale = c.endswith("_scale")
                if not isinstance(st[c], torch.Tensor) or tuple(st[c].shape) != (blocks if scale else tuple(p.shape)) or \
                        ("root" in st and st[c].dtype != (torch.float32 if scale else _F8)):
                    what = f"{st[c].dtype}, {tuple(st[c].shape)}" if isinstance(st[c], torch.Tensor) else type(st[c])
                    raise ValueError(f"loaded moments of parameter {k} ({c}: {what}) do not fit the parameter {tuple(p.shape)}")

    def load_state_dict(self, sd: dict) -> None:
        """A checkpoint that does not fit is refused and changes nothing. The state is made anew: a captured step has to be captured again."""
        self._check_loaded(sd)
        flat = self._in_order()
        like = lambda t, p, dtype: torch.empty_like(p, dtype=dtype).copy_(t.detach())  # noqa: E731
        state, counts = {}, {}
        for k, st in sd["state"].items():
            p = flat[int(k)]
            if "root" in st:                         # in their own memory order: a scale belongs to consecutive elements
                at = lambda t: t.detach().to(p.device, copy=True)  # noqa: E731
                st8 = AdamState8([at(st["exp_avg"].view(torch.uint8)).view(_F8)], [at(st["exp_avg_scale"]).contiguous()],
                                 [at(st["root"].view(torch.uint8)).view(_F8)], [at(st["root_scale"]).contiguous()])
                new = dict(zip(AdamState8._fields, (x[0] for x in st8)))
                if self._bits(p) == 32 or not all(_dense(new[c]) and _same_order(new[c], p) for c in ("exp_avg", "root")):
                    full = [torch.empty_like(new["exp_avg"], dtype=torch.float32) for _ in range(2)]
                    read_adam_state8(st8, full[:1], full[1:])
                    new = {"exp_avg": like(full[0], p, torch.float32), "exp_avg_sq": like(full[1], p, torch.float32)}
            else:
                new = {c: like(st[c], p, torch.float32) for c in ("exp_avg", "exp_avg_sq")}
            if "root" not in new and self._bits(p) == 8:
                st8 = AdamState8.zeros([p])
                write_adam_state8(st8, [new["exp_avg"]], [new["exp_avg_sq"]])
                new = dict(zip(AdamState8._fields, (x[0] for x in st8)))
            state[p] = new
            counts.setdefault(p.device, [0] * len(self._flat))[self._slot[p]] = int(st["step"])
        steps = {device: torch.tensor(c, dtype=torch.int32, device=device) for device, c in counts.items()}
        self._state, self._steps, self._lists = {}, steps, tuple([None] * len(self._flat) for _ in range(4))
        for p, new in state.items():
            self._set_state(p, new)
        for g, src in zip(self.param_groups, sd["param_groups"]):
            if isinstance(g["lr"], torch.Tensor):
                g["lr"].fill_(float(src["lr"]))
            else:
                g["lr"] = float(src["lr"])
            g["betas"], g["eps"], g["weight_decay"] = tuple(src["betas"]), float(src["eps"]), float(src["weight_decay"])

    zero_grad = SGDNesterov.zero_grad


class LinearWarmupPolyLR:
    """lr(k) with k = number of scheduler steps + 1, exactly the reference's `_step_count` arithmetic."""

    def __init__(self, optimizer: Union[SGDNesterov, AdamW], warm_iterations: int, warm_lr: float, poly_gamma: float, num_iterations: int):
        self.opt, self.warm, self.warm_lr, self.gamma, self.total = optimizer, warm_iterations, warm_lr, poly_gamma, num_iterations
        self.base_lr = optimizer.defaults["lr"]
        self._step_count = 0
        self.step()

    def get_lr(self) -> float:
        k = self._step_count
        if k - 1 < self.warm:
            return self.warm_lr + (self.base_lr - self.warm_lr) * (float(k) / float(self.warm))
        return self.base_lr * (1 - (k - self.warm) / float(self.total - self.warm)) ** self.gamma

    def step(self):
        self._step_count += 1
        self._set(self.get_lr())

    def _set(self, lr: float) -> None:
        for g in self.opt.param_groups:
            if isinstance(g["lr"], torch.Tensor):                     # a rate on the device (AdamW): what a captured step reads
                g["lr"].fill_(lr)
            else:
                g["lr"] = lr

    def state_dict(self) -> dict:
        """`_step_count` / `last_epoch` as torch's _LRScheduler keeps them (last_epoch = _step_count - 1)."""
        return {"_step_count": self._step_count, "last_epoch": self._step_count - 1, "base_lrs": [self.base_lr]}

    def load_state_dict(self, sd: dict) -> None:
        self._step_count = int(sd["_step_count"])
        self._set(self.get_lr())
