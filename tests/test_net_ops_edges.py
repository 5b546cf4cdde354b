"""Refusals and bookkeeping of the training operators (net_ops.py) without a GPU: the optimiser on CPU tensors with its
launches recorded in place of run, and the C entries' answers to arguments that no launch may see."""

import pytest
import torch

from master_doko_reinforcement_learning_amd import _native


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
