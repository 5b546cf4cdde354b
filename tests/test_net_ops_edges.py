"""Refusals and bookkeeping of the training operators (net_ops.py) without a GPU: the optimiser on CPU tensors with its
launches recorded in place of run, and the C entries' answers to arguments that no launch may see."""
import ctypes

import pytest
import torch

from master_doko_reinforcement_learning_amd import _native

INVALID = -1


@pytest.fixture
def adamw(monkeypatch):
    """(AdamW on CPU tensors, the element counts of each launch that it would have made)."""
    from master_doko_reinforcement_learning_amd import net_ops
    launches = []

    def launch(fn, index, rows, n, *args):
        got = (_native.dk_net_adamw_tensor * n).from_address(rows)
        launches.append([(t.p, t.g, t.n, t.id) for t in got])
        return 0
    monkeypatch.setattr(net_ops, "_floating", lambda t, what: net_ops._TYPES[t.dtype])
    monkeypatch.setattr(net_ops, "_INDEX", lambda t: None)
    monkeypatch.setattr(net_ops, "_launch", launch)
    return net_ops.AdamW, launches


def _params(*sizes):
    ps = [torch.zeros(n, requires_grad=True) for n in sizes]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


def test_adamw_refuses_another_number_of_elements(adamw):
    """A parameter's or gradient's memory replaced by less (or more) than the launch covers: nothing is launched."""
    AdamW, launches = adamw
    for size in (0, 10, 299, 301, 4000):
        ps = _params(300, 7)
        opt = AdamW(ps)
        opt.step()
        assert len(launches) == 1 and [t[2] for t in launches.pop()] == [300, 7]
        ps[0].data = torch.zeros(size)
        with pytest.raises(RuntimeError):      # (the old gradient)
            opt.step()
        ps[0].grad = torch.ones(size)
        with pytest.raises(RuntimeError):
            opt.step()
        ps[0].data = torch.zeros(300)          # (the other way round: a gradient of another size than its parameter)
        with pytest.raises((RuntimeError, ValueError)):
            opt.step()
        ps[0].grad = None
        opt.step()
        assert [t[2:] for t in launches.pop()] == [(7, 1)]
        ps[0].grad = torch.ones(300)
        opt.step()
        assert [t[2] for t in launches.pop()] == [300, 7]


def test_adamw_refuses_memory_that_came_to_be_shared(adamw):
    """Two parameters of a group on the same memory since the optimiser was made: two workgroups would update it at once."""
    AdamW, launches = adamw
    for shared in (lambda a: a.data, lambda a: a.data[100:].view(-1)):
        a, b, c = _params(300, 200, 9)
        opt = AdamW([a, b, c])
        opt.step()
        b.data = shared(a)[:200]
        for grad in (torch.ones(300), None, torch.ones(300)):
            a.grad = grad
            launches.clear()
            with pytest.raises(RuntimeError, match="overlap"):
                opt.step()
            assert not launches
        b.data = torch.zeros(200)
        opt.step()
        assert [(t[0], t[2]) for t in launches.pop()] == [(p.data_ptr(), p.numel()) for p in (a, b, c)]


def test_adamw_steps_with_an_empty_group(adamw):
    AdamW, launches = adamw
    p, = _params(5)
    opt = AdamW([{"params": []}, {"params": [p]}])
    opt.step()
    assert [t[2] for t in launches.pop()] == [5]


def test_adamw_load_state_dict_hooks(adamw):
    """Registered hooks run: one before, which may replace the state_dict, and one after it is loaded."""
    AdamW, _ = adamw
    ps, qs = _params(300, 7), _params(300, 7)
    opt, other = AdamW(ps, lr=0.25), AdamW(qs)
    opt.state[ps[0]]["exp_avg"].fill_(2.0)
    seen = []

    def before(o, state_dict):
        seen.append(("before", o, float(o.state[qs[0]]["exp_avg"][0])))
        state_dict["param_groups"] = [dict(g, lr=0.5) for g in state_dict["param_groups"]]   # (of its own copy)

    def replaced(o, state_dict):
        seen.append(("replaced", o, state_dict["param_groups"][0]["lr"]))
        return dict(state_dict, param_groups=[dict(g, eps=0.125) for g in state_dict["param_groups"]])
    other.register_load_state_dict_pre_hook(before)
    handle = other.register_load_state_dict_pre_hook(replaced)
    other.register_load_state_dict_post_hook(lambda o: seen.append(("after", o, float(o.state[qs[0]]["exp_avg"][0]))))
    state = opt.state_dict()
    other.load_state_dict(state)
    assert seen == [("before", other, 0.0), ("replaced", other, 0.5), ("after", other, 2.0)]
    assert other.param_groups[0]["lr"] == 0.5 and other.param_groups[0]["eps"] == 0.125 and state["param_groups"][0]["lr"] == 0.25
    handle.remove()
    other.load_state_dict(state)
    assert other.param_groups[0]["eps"] == 1e-8


def test_layer_norm_entry_refuses_strided_rows_in_place():
    """x_out is dense: over x or delta themselves only where their rows are."""
    L = _native.lib()
    buf, other = ctypes.create_string_buffer(4096), ctypes.create_string_buffer(4096)
    p, q = ctypes.addressof(buf), ctypes.addressof(other)

    def forward(x=p, x_stride=8, delta=q, delta_stride=8, x_out=p):
        return L.dk_net_layer_norm_async(x, x_stride, delta, delta_stride, 2, 8, 0, None, None, 0, 1e-5, x_out, ctypes.addressof(other) + 1024, None, None)
    assert forward(x_stride=9) == INVALID and forward(x_stride=0) == INVALID and forward(delta=None, x_stride=16) == INVALID
    assert forward(x_out=q, delta_stride=12) == INVALID and forward(x_out=q, delta_stride=0) == INVALID


def test_saved_tensors_may_come_back_with_other_strides(monkeypatch):
    """Saved-tensor hooks (torch.autograd.graph.save_on_cpu) hand back dense copies of strided rows: the backward passes
    take the strides of what they are given."""
    from master_doko_reinforcement_learning_amd import net_ops
    calls = []

    def launch(fn, index, *args):
        calls.append((fn.__name__,) + args)
        return 0
    monkeypatch.setattr(net_ops, "_floating", lambda t, what: net_ops._TYPES[t.dtype])
    monkeypatch.setattr(net_ops, "_launch", launch)
    given = {}

    def pack(t):
        copy = torch.empty(t.shape, dtype=t.dtype)
        given[copy.data_ptr()] = copy
        return copy.copy_(t)
    wide, marks = torch.zeros(6, 50), torch.ones(6, 47, dtype=torch.bool)
    for mask, strides in ((None, (0,)), (marks[:, 3:43], (40,)), (marks[0, :40], (0,)), (marks[0, :40].expand(6, 40), (0, 40))):
        x = wide[:, 5:45].requires_grad_()
        for hooked in (False, True):
            with torch.autograd.graph.saved_tensors_hooks(pack if hooked else lambda t: t, lambda t: t):
                got = net_ops.token_logprobs(x, torch.zeros(6, dtype=torch.int64), mask=mask)
            torch.autograd.grad(got.logprobs.sum(), x)
            name, logits, stride, rows, vocab, _, m, mask_stride = calls.pop()[:8]
            assert name == "dk_net_token_logprobs_bwd_async" and (rows, vocab) == (6, 40) and stride == (40 if hooked else 50)
            if hooked:
                assert logits in given and (m is None) == (mask is None) and (m is None or m in given) and mask_stride in strides
            elif mask is not None:
                assert m == mask.data_ptr() and mask_stride == (0 if mask.dim() == 1 else mask.stride(0))
    x, w = wide[:, 5:45].requires_grad_(), torch.ones(40)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        h = net_ops.layer_norm(x, w)
    torch.autograd.grad(h.sum(), x)
    name, _, dh_stride, _, _, rows, stride = calls.pop()[:7]
    assert name == "dk_net_layer_norm_bwd_async" and rows in given and (dh_stride, stride) == (40, 40)


def test_token_logprobs_entry_refuses_the_gradient_over_the_logits():
    """The tokens' logits are read again after the row's gradients are written."""
    L = _native.lib()
    buf, other = ctypes.create_string_buffer(4096), ctypes.create_string_buffer(4096)
    x, p = ctypes.addressof(buf), ctypes.addressof(other)
    assert L.dk_net_token_logprobs_bwd_async(x, 8, 1, 8, 0, None, 0, 1.0, p, 1, p, p, p, p, None, x, None) == INVALID
