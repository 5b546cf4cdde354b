"""The training operators' refusals, without a GPU: the Python entry points need GPU tensors, and the C entries answer
bad arguments with DK_E_INVALID before anything is launched."""
import ctypes

import pytest
import torch

from master_doko_reinforcement_learning_amd import _native

INVALID = -1


def test_entry_points_need_the_gpu():
    from master_doko_reinforcement_learning_amd import AdamW, layer_norm, token_logprobs
    x = torch.zeros(2, 8)
    for bad in (lambda: layer_norm(x), lambda: token_logprobs(x), lambda: AdamW([x.requires_grad_()]), lambda: layer_norm([1.0])):
        with pytest.raises(ValueError):
            bad()


def test_package_does_not_import_torch():
    import subprocess
    import sys
    code = "import sys, master_doko_reinforcement_learning_amd as d; assert 'torch' not in sys.modules; d.layer_norm; assert 'torch' in sys.modules"
    subprocess.run([sys.executable, "-c", code], check=True)
    import master_doko_reinforcement_learning_amd as d
    with pytest.raises(AttributeError):
        d.no_such_name


def test_layer_norm_entries_refuse():
    L = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)

    def forward(x=p, delta=None, rows=1, d=8, type=0, wtype=0, x_out=None, h=p):
        return L.dk_net_layer_norm_async(x, d, delta, d, rows, d, type, None, None, wtype, 1e-5, x_out, h, None, None)
    for bad in (dict(type=3), dict(type=-1), dict(wtype=1), dict(type=1, wtype=2), dict(d=0), dict(d=16385), dict(delta=p), dict(x=None), dict(h=None), dict(rows=1 << 40)):
        assert forward(**bad) == INVALID, bad
    assert forward(rows=0, x=None, h=None) == 0

    def backward(dh=p, x=p, stats=p, rows=1, d=8, type=0, wtype=0, dx=p, dw=p, ws=p, size=4096):
        return L.dk_net_layer_norm_bwd_async(dh, d, None, 0, x, d, stats, rows, d, type, None, wtype, dx, dw, None, ws, size, None)
    for bad in (dict(dh=None), dict(x=None), dict(stats=None), dict(dx=None), dict(ws=None), dict(size=3), dict(type=7), dict(wtype=2), dict(d=0)):
        assert backward(**bad) == INVALID, bad
    assert backward(rows=0, dw=None, ws=None, dh=None, x=None, stats=None, dx=None) == 0
    assert L.dk_net_layer_norm_bwd_workspace(1000, 160, 0) >= 2 * 160 * 4


def test_token_logprobs_entries_refuse():
    L = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)

    def forward(x=p, rows=1, vocab=8, type=0, temperature=1.0, tokens=p, n=1, top=0, lp=p, tl=None, tt=None):
        return L.dk_net_token_logprobs_async(x, vocab, rows, vocab, type, None, 0, temperature, tokens, n, top, lp, None, None, tl, tt, None, 0, None)
    for bad in (dict(type=4), dict(vocab=0), dict(n=65), dict(top=33), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(temperature=1e-40), dict(temperature=2e30), dict(x=None), dict(tokens=None), dict(lp=None), dict(top=1), dict(top=1, tl=p), dict(rows=1 << 33)):
        assert forward(**bad) == INVALID, bad
    assert forward(rows=0, x=None) == 0

    def backward(x=p, rows=1, vocab=8, type=0, temperature=1.0, tokens=p, n=1, lp=p, lse=p, ent=p, dx=p):
        return L.dk_net_token_logprobs_bwd_async(x, vocab, rows, vocab, type, None, 0, temperature, tokens, n, lp, lse, ent, None, None, dx, None)
    for bad in (dict(type=4), dict(vocab=0), dict(n=65), dict(temperature=-1.0), dict(temperature=1e-40), dict(x=None), dict(tokens=None), dict(lp=None), dict(lse=None), dict(ent=None), dict(dx=None)):
        assert backward(**bad) == INVALID, bad
    assert backward(rows=0, x=None) == 0


def test_adamw_entry_refuses():
    L = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)

    def step(rows=((p, p, 8, 0, 0),), type=0, bits=32, m=p, v=p, ms=None, step=p, factors=p, b1=0.9, b2=0.99, eps=1e-8):
        t = (_native.dk_net_adamw_tensor * max(1, len(rows)))(*rows)
        return L.dk_net_adamw_async(ctypes.addressof(t), len(rows), type, bits, m, v, ms, ms, None, step, factors, 1e-3, None, b1, b2, eps, 0.0, None)
    for bad in (dict(type=3), dict(bits=16), dict(bits=8), dict(m=None), dict(v=None), dict(step=None), dict(factors=None), dict(b1=1.0), dict(b2=-0.1),
                dict(b1=float("nan")), dict(eps=-1.0), dict(rows=((None, p, 8, 0, 0),)), dict(rows=((p, None, 8, 0, 0),)), dict(rows=((p, p, 1 << 50, 0, 0),))):
        assert step(**bad) == INVALID, bad
    assert step(rows=()) == 0


def test_launches_go_to_the_tensors_device(monkeypatch):
    """A tensor on another device than the current one: its device is current during the call, and the stream is its own."""
    import contextlib

    from master_doko_reinforcement_learning_amd import net_ops
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        current.append(index)
        yield
        current.pop()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[-1])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(net_ops, "_raw_stream", lambda i: 100 + i)
    entry = lambda *a: seen.append((current[-1],) + a) or 0  # noqa: E731
    assert net_ops._launch(entry, 0, "x") == 0 and net_ops._launch(entry, 3, "y") == 0
    assert seen == [(0, "x", 100), (3, "y", 103)] and current == [0]
