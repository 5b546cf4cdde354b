"""The operators of a training step on the GPU: LayerNorm with the residual add before it, log
probabilities of given tokens with entropy and top alternatives, and AdamW over many tensors at once.

Each is a HIP kernel behind the C-ABI (dk_net_layer_norm_*, dk_net_token_logprobs_*,
dk_net_adamw_async; csrc/train_*_kernels.h) on torch's current stream of the tensors' device, and the
first two are differentiable (once, in reverse mode).  f32, bf16 and f16; sums and statistics are f32.  There is no CPU
fallback.  DokoAzNet.loss / DokoImpiNet.loss are built on the first two, NetTrainer on all three.
"""
import collections
import itertools
import math
import operator
from typing import NamedTuple, Optional

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _native

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # enum dk_net_type
NORM_MAX_D, VOCAB_MAX, TOKENS_MAX, TOP_MAX, ADAMW_BLOCK = 16384, (1 << 31) - 1, 64, 32, 256


def _check(rc, what):
    if rc != 0:
        raise RuntimeError("doko_amd %s kernel error %d" % (what, rc))


# torch's current stream of a device as an integer (the public call makes a Stream object each time, 2 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _launch(fn, index, *args):
    """fn(*args, stream) on torch's current stream of device `index`, with that device current."""
    if index == torch.cuda.current_device():
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return fn(*args, _raw_stream(index))


def _rows(t):
    """t as rows over its last dimension: (a tensor with that memory, elements between rows).
    Copies only what has no such view."""
    if t.is_contiguous():
        return t, t.shape[-1]
    r = t.reshape(-1, t.shape[-1])
    if r.stride(1) != 1 and r.shape[1] > 1:
        r = r.contiguous()
    return r, r.stride(0)


def _floating(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s: a tensor on the GPU is needed" % what)
    if t.dtype not in _TYPES:
        raise ValueError("%s: float32, bfloat16 or float16 is needed, got %s" % (what, t.dtype))
    return _TYPES[t.dtype]


def _no_tangents(what, *tensors):
    """Raises for a forward-mode dual tensor: the kernels would read its values and drop its tangent."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("%s has no forward-mode derivative" % what)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------- layer norm
def _dense_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _norm_forward(x, delta, weight, bias, eps, stats):
    d = x.shape[-1]
    rows = x.numel() // d
    xr, xs = _rows(x)
    dr, ds = _rows(delta) if delta is not None else (None, 0)
    h = _dense_like(x)
    new = _dense_like(x) if delta is not None else None
    st = x.new_empty((rows, 2), dtype=torch.float32) if stats else None
    w = weight if weight is not None else bias
    _check(_launch(_native.lib().dk_net_layer_norm_async, x.get_device(), xr.data_ptr(), xs, _ptr(dr), ds, rows, d, _TYPES[x.dtype],
                   _ptr(weight), _ptr(bias), _TYPES[w.dtype] if w is not None else 0, eps, _ptr(new), h.data_ptr(), _ptr(st)),
           "layer norm")
    return new, h, st, xr


def _norm_backward(ctx, *grads):
    dres, dh = (None, grads[0]) if len(grads) == 1 else grads
    need_x, need_delta, need_w, need_b, _ = ctx.needs_input_grad
    if dh is None:
        return (dres if need_x else None), (dres if need_delta else None), None, None, None
    x, st, weight = ctx.saved_tensors
    wdtype = weight.dtype if weight is not None else ctx.wdtype
    rows, d, kind = st.shape[0], x.shape[-1], _TYPES[x.dtype]
    xr, xs = _rows(x)
    gr, gs = _rows(dh)
    rr, rs = _rows(dres) if dres is not None else (None, 0)
    dx = _dense_like(x)
    dw = x.new_empty(d, dtype=wdtype) if need_w else None
    db = x.new_empty(d, dtype=wdtype) if need_b else None
    L = _native.lib()
    size = L.dk_net_layer_norm_bwd_workspace(rows, d, kind) if need_w or need_b else 0
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _check(_launch(L.dk_net_layer_norm_bwd_async, x.get_device(), gr.data_ptr(), gs, _ptr(rr), rs, xr.data_ptr(), xs, st.data_ptr(),
                   rows, d, kind, _ptr(weight), _TYPES[wdtype], dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), size),
           "layer norm backward")
    if dx.shape != ctx.shape:   # (x was copied into rows)
        dx = dx.view(ctx.shape)
    return (dx if need_x else None), (dx if need_delta else None), dw, db, None


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, weight, bias, eps):
        new, h, st, xr = _norm_forward(x, delta, weight, bias, eps, True)
        ctx.shape, ctx.wdtype = x.shape, torch.float32 if bias is None else bias.dtype
        ctx.save_for_backward(xr if new is None else new, st, weight)
        ctx.set_materialize_grads(False)
        return h if new is None else (new, h)

    @staticmethod
    def backward(ctx, *grads):   # (the check against a second derivative only where one is asked for: 4 us)
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, *grads)


def layer_norm(x, weight=None, bias=None, eps=1e-5, delta=None):
    """LayerNorm over the last dimension (at most 16384 columns), any leading dimensions and row stride.

    With `delta` (x's shape and dtype) the residual stream moves on first: returns (x + delta, LayerNorm of
    it), both differentiable; the sum is rounded to the dtype, and it is the rounded one that is normalised.
    weight / bias: [columns] in x's dtype or float32 (both the same), or None for 1 / 0."""
    _floating(x, "layer_norm")
    if x.dim() == 0 or not 0 < x.shape[-1] <= NORM_MAX_D:
        raise ValueError("layer_norm: 1 to %d columns, got %s" % (NORM_MAX_D, tuple(x.shape)))
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError("layer_norm: eps %r" % (eps,))
    if delta is not None and (not isinstance(delta, torch.Tensor) or delta.shape != x.shape or delta.dtype != x.dtype or delta.device != x.device):
        raise ValueError("layer_norm: delta has x's shape, dtype and device")
    for t in (weight, bias):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.device != x.device or t.shape != x.shape[-1:] or t.dtype not in (x.dtype, torch.float32):
            raise ValueError("layer_norm: weight and bias are [%d] tensors in %s or float32 on %s" % (x.shape[-1], x.dtype, x.device))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias differ in dtype")
    _no_tangents("layer_norm", x, delta, weight, bias)
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, delta, weight, bias)):
        return _LayerNorm.apply(x, delta, weight, bias, eps)
    new, h, _, _ = _norm_forward(x, delta, weight, bias, eps, False)
    return h if new is None else (new, h)


# ------------------------------------------------------------------------------- log probabilities
class TokenLogprobs(NamedTuple):
    """token_logprobs' answer: f32 log probabilities in the tokens' shape, the rows' entropy, and the
    `top` largest log probabilities of each row with their tokens (None where top is 0)."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _mask_rows(mask):
    """A mask as _rows has it; one of a single dimension goes for every row."""
    return (None, 0) if mask is None else (mask.contiguous(), 0) if mask.dim() == 1 else _rows(mask)


def _logp_forward(logits, tokens, mask, temperature, top, stats):
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    rows = logits.numel() // vocab
    xr, xs = _rows(logits)
    mr, ms = _mask_rows(mask)
    n = 0 if tokens is None else 1 if tokens.dim() == len(lead) else tokens.shape[-1]
    f32 = torch.float32
    logprobs = None if tokens is None else logits.new_empty(tokens.shape, dtype=f32)
    entropy = logits.new_empty(lead, dtype=f32)
    st = logits.new_empty((rows, 2), dtype=f32) if stats else None
    tl = logits.new_empty(lead + (top,), dtype=f32) if top else None
    tt = logits.new_empty(lead + (top,), dtype=torch.int64) if top else None
    L, kind = _native.lib(), _TYPES[logits.dtype]
    size = L.dk_net_token_logprobs_workspace(rows, vocab, kind, top)
    ws = logits.new_empty(size, dtype=torch.uint8) if size else None
    _check(_launch(L.dk_net_token_logprobs_async, logits.get_device(), xr.data_ptr(), xs, rows, vocab, kind, _ptr(mr), ms, temperature,
                   _ptr(tokens), n, top, _ptr(logprobs), entropy.data_ptr(), _ptr(st), _ptr(tl), _ptr(tt), _ptr(ws), size),
           "token log probabilities")
    return logprobs, entropy, st, tl, tt, (xr, mr, n)


def _logp_backward(ctx, dlogp, dent, _tl, _tt):
    if dlogp is None and dent is None:
        return None, None, None, None, None
    x, tokens, mask, logprobs, st, entropy = ctx.saved_tensors
    xr, xs = _rows(x)   # (saved tensors may come back with other strides: hooks copy them)
    mr, ms = _mask_rows(mask)
    dlogp = None if dlogp is None else dlogp.contiguous()
    dent = None if dent is None else dent.contiguous()
    dx = x.new_empty(ctx.shape)
    _check(_launch(_native.lib().dk_net_token_logprobs_bwd_async, x.get_device(), xr.data_ptr(), xs, st.shape[0], x.shape[-1],
                   _TYPES[x.dtype], _ptr(mr), ms, ctx.temperature, _ptr(tokens), ctx.n, _ptr(logprobs), st.data_ptr(),
                   entropy.data_ptr(), _ptr(dlogp), _ptr(dent), dx.data_ptr()), "token log probabilities backward")
    return dx, None, None, None, None


_logp_backward_once = torch.autograd.function.once_differentiable(_logp_backward)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, top):
        logprobs, entropy, st, tl, tt, (xr, mr, n) = _logp_forward(logits, tokens, mask, temperature, top, True)
        ctx.save_for_backward(xr, tokens, mr, logprobs, st, entropy)
        ctx.n, ctx.temperature, ctx.shape = n, temperature, logits.shape
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(tl, tt)
        return logprobs, entropy, tl, tt

    @staticmethod
    def backward(ctx, *grads):
        return (_logp_backward_once if torch.is_grad_enabled() else _logp_backward)(ctx, *grads)


def token_logprobs(logits, tokens=None, mask=None, temperature=1.0, top=0):
    """Log probabilities of given tokens under softmax(logits / temperature), with the rows' entropy and their
    `top` (at most 32) largest alternatives; differentiable in the logits through logprobs and entropy.

    logits [..., vocab]; tokens int64 or int32 [...] or [..., n] with n <= 64; a negative one is padding (log
    probability 0, no gradient), one >= vocab gives NaN and no gradient.  mask: bool [..., vocab] or [vocab],
    True for what is allowed; a token that is not has log probability -inf and no gradient, and what a masked
    logit holds is not looked at (nor has one a gradient whose log probability is below float32's range).  A row with nothing allowed has entropy 0.  Alternatives are ordered by
    logit, equal ones by index; -1 (and -inf) behind the last allowed one."""
    _floating(logits, "token_logprobs")
    if logits.dim() == 0 or not 0 < logits.shape[-1] <= VOCAB_MAX:   # (the entries take 32 bits of it)
        raise ValueError("token_logprobs: a vocabulary of 1 to %d, got logits %s" % (VOCAB_MAX, tuple(logits.shape)))
    lead = logits.shape[:-1]
    if tokens is not None:
        if not isinstance(tokens, torch.Tensor) or tokens.device != logits.device or tokens.dtype not in (torch.int64, torch.int32):
            raise ValueError("token_logprobs: tokens are int64 or int32 on the logits' device")
        if tokens.shape != lead and not (tokens.dim() == len(lead) + 1 and tokens.shape[:-1] == lead and tokens.shape[-1] <= TOKENS_MAX):
            raise ValueError("token_logprobs: tokens %s do not go with logits %s (at most %d a row)"
                             % (tuple(tokens.shape), tuple(logits.shape), TOKENS_MAX))
        tokens = tokens.long().contiguous()
    if mask is not None and (not isinstance(mask, torch.Tensor) or mask.device != logits.device or mask.dtype != torch.bool
                             or mask.shape not in (logits.shape, logits.shape[-1:])):
        raise ValueError("token_logprobs: mask is bool on the logits' device, in their shape or [%d]" % logits.shape[-1])
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e30:
        raise ValueError("token_logprobs: temperature %r (1e-6 to 1e30)" % (temperature,))
    if not 0 <= top <= TOP_MAX:
        raise ValueError("token_logprobs: top %r (0 to %d)" % (top, TOP_MAX))
    _no_tangents("token_logprobs", logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, mask, temperature, top))
    logprobs, entropy, _, tl, tt, _ = _logp_forward(logits, tokens, mask, temperature, top, False)
    return TokenLogprobs(logprobs, entropy, tl, tt)


# ------------------------------------------------------------------------------- AdamW
_GRAD, _DTYPE = operator.attrgetter("grad"), operator.attrgetter("dtype")
_DENSE, _NUMEL, _PTR = torch.Tensor.is_contiguous, torch.Tensor.numel, torch.Tensor.data_ptr
_INDEX = torch.Tensor.get_device   # (-1 on the CPU)
_ROW = np.dtype([("p", np.uint64), ("g", np.uint64), ("n", np.uint64), ("block", np.uint64), ("id", np.uint64)])


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay, bias-corrected moments) with one pass over all tensors of a group.

    state_bits 32: f32 moments.  state_bits 8: e4m3 codes of exp_avg and of sqrt(exp_avg_sq) with one f32
    scale for each 256 elements of a tensor.  master_weights: bf16 / f16 parameters are rounded copies of
    f32 weights that the optimiser keeps; a parameter that was written to since the last step (a loaded
    state_dict) is taken over into its master first.  step() sees that by the parameter's version counter, which
    a write through .data does not raise, and a captured step does not look: refresh_masters() takes over what was
    written in such ways, and before a capture.  lr may be a one-element f32 tensor on the GPU.

    A group's parameters share one dtype and device, are dense and do not overlap.  The states lie in flat buffers
    (`buffers`, one dict a group; each parameter at a multiple of 256 elements) and state[p] holds views of
    them; `step` counts on the device for each parameter, so step() may be captured into a graph
    (lr as a float is captured as it is).  step() raises the parameters' version counters, by which the networks'
    fused forwards notice new weights; the replay of a captured one does not."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master_weights=False):
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits %r (8 or 32)" % (state_bits,))
        self.state_bits, self.master_weights = state_bits, bool(master_weights)
        self.buffers, self._tables = [], []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @torch.no_grad()
    def __getstate__(self):   # (a copy or a pickle, which knows no e4m3: the codes as bytes; the buffers are laid out anew)
        self._take_over_written()
        state = super().__getstate__()
        state["state"] = {p: {k: v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v for k, v in st.items()}
                          for p, st in state["state"].items()}
        return {**state, "state_bits": self.state_bits, "master_weights": self.master_weights}

    @torch.no_grad()
    def __setstate__(self, state):
        super().__setstate__(state)
        old, self.state, self.buffers, self._tables = self.state, collections.defaultdict(dict), [], []
        for group in self.param_groups:
            self._lay_out(group)
            for p in group["params"]:
                for k, v in self.state[p].items():
                    v.copy_(old[p][k].view(v.dtype) if v.dtype == torch.float8_e4m3fn else old[p][k])

    @torch.no_grad()
    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._lay_out(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def _lay_out(self, group):
        params = group["params"]
        _hyper(group)
        for p in params:
            _floating(p, "AdamW")
            if p.dtype != params[0].dtype or p.device != params[0].device or not p.is_contiguous():
                raise ValueError("AdamW: a group's parameters are dense and share one dtype and device")
        if _overlap(params):
            raise ValueError("AdamW: a group's parameters overlap, or one is given twice")
        master = self.master_weights and bool(params) and params[0].dtype != torch.float32
        dev = params[0].device if params else None
        table = np.zeros(len(params), _ROW)
        blocks = 0
        for i, p in enumerate(params):
            table[i] = (p.data_ptr(), 0, p.numel(), blocks, i)
            blocks += -(-p.numel() // ADAMW_BLOCK)
        b = {"step": torch.zeros(len(params), dtype=torch.int32, device=dev)}
        for k in ("exp_avg", "exp_avg_sq"):
            if self.state_bits == 8:
                b[k] = torch.zeros(blocks * ADAMW_BLOCK, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
                b[k + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=dev)
            else:
                b[k] = torch.zeros(blocks * ADAMW_BLOCK, dtype=torch.float32, device=dev)
        if master:
            b["master"] = torch.zeros(blocks * ADAMW_BLOCK, dtype=torch.float32, device=dev)
        for i, p in enumerate(params):
            lo, n = int(table[i]["block"]), p.numel()
            st = self.state[p] = {"step": b["step"][i]}
            for k in b:
                if k.endswith("_scale"):
                    st[k] = b[k][lo:lo + -(-n // ADAMW_BLOCK)]
                elif k != "step":
                    st[k] = b[k][lo * ADAMW_BLOCK:lo * ADAMW_BLOCK + n].view(p.shape)
            if master:
                st["master"].copy_(p)
        # (scratch of a step: the tensors' factors; and the parameters' versions that the masters go with)
        self.buffers.append(b)
        self._tables.append({"rows": table, "sizes": list(map(_NUMEL, params)), "memory": list(map(_PTR, params)),
                             "dtype": params[0].dtype if params else None, "device": dev,
                             "factors": torch.empty(3 * max(1, len(params)), dtype=torch.float32, device=dev),
                             "versions": [p._version for p in params] if master else None})

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group, b, t in zip(self.param_groups, self.buffers, self._tables):
            self._step_group(group, b, t)
        return loss

    def _step_group(self, group, b, t):
        dtype, device = t["dtype"], t["device"]
        lr, d_lr = _hyper(group)
        params, sizes, known, at = group["params"], t["sizes"], t["memory"], None
        grads = list(map(_GRAD, params))
        if not all(map(operator.is_not, grads, itertools.repeat(None))):
            at = [i for i, g in enumerate(grads) if g is not None]
            params, grads, sizes, known = ([u[i] for i in at] for u in (params, grads, sizes, known))
        if not params:
            return
        if d_lr is not None and d_lr.device != device:
            raise ValueError("AdamW: lr lies on another device than its group")
        # (checked anew each step, in maps: a network has a hundred tensors, and the step takes 20 us on the GPU)
        if (list(map(_NUMEL, params)) != sizes or set(map(_DTYPE, params)) != {dtype} or set(map(_INDEX, params)) != {device.index}
                or not all(map(_DENSE, params))):
            raise RuntimeError("AdamW: a parameter was moved, cast, resized or restrided since the optimiser was made")
        try:
            if set(map(_DTYPE, grads)) != {dtype} or list(map(_NUMEL, grads)) != sizes:
                raise RuntimeError
            if not all(map(_DENSE, grads)):   # (raises for a sparse one)
                grads = [g.contiguous() for g in grads]
        except RuntimeError:
            raise ValueError("AdamW: gradients are dense and of the parameters' sizes and dtype") from None
        versions = t["versions"]
        if versions is not None:
            self._take_over(t, [(i, p) for i, p in zip(at or range(len(params)), params) if versions[i] != p._version])
        n = len(params)
        rows = t["rows"] if at is None else t["rows"][at]
        memory = list(map(_PTR, params))
        if memory != known:   # (new memory, through p.data: looked at as the first was)
            if _overlap(group["params"]):
                raise RuntimeError("AdamW: a group's parameters overlap since the optimiser was made")
            t["rows"]["p"][slice(None) if at is None else at] = rows["p"] = memory
            for i, m in zip(at or range(n), memory):
                t["memory"][i] = m
        rows["g"] = np.fromiter(map(_PTR, grads), np.uint64, n)
        b1, b2 = group["betas"]
        _check(_launch(_native.lib().dk_net_adamw_async, device.index, rows.ctypes.data, n, _TYPES[dtype], self.state_bits,
                       b["exp_avg"].data_ptr(), b["exp_avg_sq"].data_ptr(), _ptr(b.get("exp_avg_scale")),
                       _ptr(b.get("exp_avg_sq_scale")), _ptr(b.get("master")), b["step"].data_ptr(), t["factors"].data_ptr(),
                       lr, _ptr(d_lr), b1, b2, group["eps"], group["weight_decay"]), "AdamW")
        # the networks' split weights are cached by the parameters' versions
        torch.autograd.graph.increment_version(params)
        if versions is not None:
            for i, p in zip(at or range(n), params):
                versions[i] = p._version

    @torch.no_grad()
    def refresh_masters(self):
        """Takes every parameter whose values are not its rounded master's over into the master: written to through
        .data, between the replays of a captured step, or before one is captured (not within a capture itself)."""
        for group, t in zip(self.param_groups, self._tables):
            if t["versions"] is not None:
                self._take_over(t, list(enumerate(group["params"])))

    def _take_over_written(self):   # (what step() would see)
        for group, t in zip(self.param_groups, self._tables):
            if t["versions"] is not None:
                self._take_over(t, [(i, p) for i, p in enumerate(group["params"]) if t["versions"][i] != p._version])

    @torch.no_grad()
    def state_dict(self):
        """torch.optim.Optimizer.state_dict; the masters in it go with the parameters as they are."""
        self._take_over_written()
        return super().state_dict()

    def _take_over(self, t, written):
        """The masters of the parameters `written`, (place in the group, parameter) each.  One whose values are its rounded
        master's keeps that, which holds more of them: its version counter may be raised by others than writers."""
        if not written:
            return
        with torch.cuda.device(t["device"]):
            if torch.cuda.is_current_stream_capturing():   # (each replay would round the masters)
                raise RuntimeError("AdamW: a parameter was written to since the last step: refresh_masters() before the capture")
        for i, p in written:
            master, values = self.state[p]["master"].view(-1), p.detach().reshape(-1).to(t["device"])
            if values.numel() != master.numel():
                raise RuntimeError("AdamW: a parameter was resized since the optimiser was made")
            torch.where((master.to(t["dtype"]) == values).all(), master, values, out=master)
            t["versions"][i] = p._version

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes over the states of a state_dict() of the same parameters, into the buffers that are there
        (also torch.optim.AdamW's, where state_bits is 32); runs the hooks registered for it."""
        state_dict = dict(state_dict)   # (a hook may write to it)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("AdamW: the state_dict has other parameter groups")
        if any(g.get("amsgrad") or g.get("maximize") for g in groups):
            raise ValueError("AdamW: the state_dict is of another update (amsgrad, maximize)")
        todo = []
        for mine, theirs in zip(self.param_groups, groups):
            for p, key in zip(mine["params"], theirs["params"]):
                st = state_dict["state"].get(key)
                for k, own in self.state[p].items():
                    if st is None or (k == "master" and k not in st):   # (not stepped yet: as at the start)
                        todo.append((own, p if k == "master" else None))
                        continue
                    v = st.get(k)
                    f8 = torch.float8_e4m3fn
                    if not isinstance(v, torch.Tensor) or v.shape != own.shape or (own.dtype == f8) != (v.dtype == f8):
                        raise ValueError("AdamW: the state_dict's %s does not fit (state_bits %d)" % (k, self.state_bits))
                    todo.append((own, v))
        for mine, theirs in zip(self.param_groups, groups):
            lr = mine["lr"]
            mine.update({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in theirs.items() if k != "params"})
            if isinstance(lr, torch.Tensor):   # (a captured step reads it)
                lr.copy_(torch.as_tensor(mine["lr"]).reshape(lr.shape))
                mine["lr"] = lr
        for own, v in todo:
            if v is None:
                own.view(torch.uint8 if own.dtype == torch.float8_e4m3fn else own.dtype).zero_()
            else:
                own.copy_(v)
        for t, g in zip(self._tables, self.param_groups):
            if t["versions"] is not None:
                t["versions"] = [p._version for p in g["params"]]
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)


def _overlap(params):
    """Whether two parameters share memory: a group's are updated side by side."""
    spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
    return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


def _hyper(group):
    """A group's learning rate as (float, device tensor or None); raises where a hyperparameter is out of range."""
    lr, (b1, b2) = group["lr"], group["betas"]
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and group["eps"] >= 0.0 and group["weight_decay"] >= 0.0):
        raise ValueError("AdamW: betas %r, eps %r or weight_decay %r out of range" % (group["betas"], group["eps"], group["weight_decay"]))
    if isinstance(lr, torch.Tensor):
        if lr.numel() != 1 or (lr.is_cuda and lr.dtype != torch.float32):
            raise ValueError("AdamW: lr as a tensor is one float32 value")
        return (0.0, lr) if lr.is_cuda else (float(lr), None)
    if not lr >= 0.0:
        raise ValueError("AdamW: lr %r" % (lr,))
    return float(lr), None
