"""The training operators (net_ops.py) on the GPU where their formulas leave float32's range, where a caller writes to
what an optimiser keeps a copy of, and where a call has to be refused."""
import copy
import math

import pytest
import torch

import net_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)


# (39: a row in 16 lanes' registers; 700: a row by a wave; 9001: by a workgroup)
@pytest.mark.parametrize("vocab", [39, 700, 9001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("temperature", [0.4, 0.99, 1.0, 1.5])
def test_gradient_of_the_types_lowest_values(vocab, dtype, temperature):
    """Additive masks of the type's lowest value: (v - max) / T leaves float32, and the entry, whose probability is 0,
    takes no gradient, with or without one of the entropy."""
    from master_doko_reinforcement_learning_amd import token_logprobs
    g = _gen(vocab)
    low = torch.finfo(dtype).min
    x = _randn(g, 6, vocab, dtype=dtype, scale=2.5)
    gone = torch.zeros(6, vocab, dtype=torch.bool, device=DEV)
    gone[0, ::3], gone[1, 1:], gone[2, 8:], gone[4, :vocab - 2] = True, True, True, True
    t = torch.tensor([[1, 2], [0, 0], [7, 3], [4, 4], [vocab - 1, -1], [0, vocab - 1]], device=DEV)
    x = torch.where(gone, low, x)
    dl = _randn(g, 6, 2)
    for de in (None, torch.full((6,), 4.0, device=DEV), torch.full((6,), -0.25, device=DEV)):
        leaf = x.detach().requires_grad_()
        got = token_logprobs(leaf, t, temperature=temperature)
        outs, grads = ([got.logprobs], [dl]) if de is None else ([got.logprobs, got.entropy], [dl, de])
        dx, = torch.autograd.grad(outs, [leaf], grads)
        want, _, _ = ref.logp(x.double(), t, None, temperature, dl.double(), None if de is None else de.double(), dtype)
        assert ref.off(dx, *want["dlogits"]) <= 1
        assert not dx[gone].any()
        if de is not None:   # the entropy's gradient alone
            leaf = x.detach().requires_grad_()
            dx, = torch.autograd.grad(token_logprobs(leaf, temperature=temperature).entropy, leaf, de)
            want, _, _ = ref.logp(x.double(), t[:, :0], None, temperature, None, de.double(), dtype)
            assert ref.off(dx, *want["dlogits"]) <= 1 and not dx[gone].any()
    if dtype == F32 and temperature < 1:
        # a token whose log probability is below float32's range has -inf and no gradient; the row's others stay
        under = t.clone()
        under[0, 1] = 0
        leaf = x.detach().requires_grad_()
        got = token_logprobs(leaf, under, temperature=temperature)
        dx, = torch.autograd.grad(got.logprobs, leaf, dl)
        assert got.logprobs[0, 1] == -math.inf
        one = t.clone()
        one[0, 1] = -1
        leaf = x.detach().requires_grad_()
        want, = torch.autograd.grad(token_logprobs(leaf, one, temperature=temperature).logprobs, leaf, dl)
        assert torch.equal(dx, want)
    # a gradient that is not finite shows in its row (loss scaling looks for it), and in no other
    bad = dl.clone()
    bad[2, 0] = math.inf
    leaf = x.detach().requires_grad_()
    dx, = torch.autograd.grad(token_logprobs(leaf, t, temperature=temperature).logprobs, leaf, bad)
    assert not dx[2].isfinite().all() and dx[[0, 1, 3, 4, 5]].isfinite().all()


@pytest.mark.parametrize("vocab", [39, 700, 9001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_disallowed_entries_of_nan_rows_take_no_gradient(vocab, dtype):
    """A NaN or +inf in an allowed entry makes its row NaN; masked entries and those of -inf still take nothing, also where
    they are among the row's tokens."""
    from master_doko_reinforcement_learning_amd import token_logprobs
    g = _gen(vocab)
    x = _randn(g, 4, vocab, dtype=dtype)
    mask = torch.rand(4, vocab, generator=g, device=DEV) < 0.5
    mask[:, 0], mask[:, 1], mask[:, 2], mask[:, 3] = True, False, True, False
    x[0, 0], x[1, 0], x[2, 0] = math.nan, math.inf, -math.inf
    x[:, 2] = -math.inf
    x[:, 3] = math.nan
    t = torch.tensor([[1, 2, 4, 1]] * 4, device=DEV)
    leaf = x.requires_grad_()
    got = token_logprobs(leaf, t, mask=mask)
    dx, = torch.autograd.grad([got.logprobs, got.entropy], [leaf], [_randn(g, 4, 4), _randn(g, 4)])
    dead = ~mask | (x.detach() == -math.inf)
    assert not dx[dead].any()
    assert dx[:2][~dead[:2]].isnan().all() and dx[2:].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [39, 700, 3000, 9001, 40000])
def test_results_do_not_depend_on_a_common_offset(vocab, dtype):
    """Sums are of differences from the row's maximum: a common offset that leaves the logits exact leaves every bit, and a
    row of the type's lowest value alone is the uniform distribution."""
    from master_doko_reinforcement_learning_amd import token_logprobs
    g = _gen(vocab)
    # whole numbers of 0 to 15, f32: and 2^20, bf16: and 128 (8 bits hold 128 to 143)
    x = torch.randint(0, 16, (5, vocab), generator=g, device=DEV).to(dtype)
    t = torch.randint(0, vocab, (5, 3), generator=g, device=DEV)
    dl, de = _randn(g, 5, 3), _randn(g, 5)
    outs = []
    for shift in (0.0, 2.0 ** 20 if dtype == F32 else 128.0, -2.0 ** 20 if dtype == F32 else -143.0):
        z = x + shift
        assert torch.equal(z.double() - shift, x.double())
        leaf = z.requires_grad_()
        got = token_logprobs(leaf, t, temperature=0.75, top=4)
        dx, = torch.autograd.grad([got.logprobs, got.entropy], [leaf], [dl, de])
        outs.append([o.detach() for o in got] + [dx])
    for o in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(o, outs[0]))
    for temperature in (0.5, 1.0):
        low = torch.full((2, vocab), torch.finfo(dtype).min, device=DEV, dtype=dtype, requires_grad=True)
        got = token_logprobs(low, t[:2], temperature=temperature)
        # log of a sum of `vocab` ones: whole numbers below 2^24 add up exactly, so one rounding of the logarithm (and 3 steps of it)
        size = math.log(vocab)
        assert (got.logprobs.detach().double() + size).abs().max() <= 4 * ref.U * size
        assert (got.entropy.detach().double() - size).abs().max() <= 4 * ref.U * size
        dx, = torch.autograd.grad(got.logprobs.sum(), low)
        n = torch.zeros(2, vocab, device=DEV, dtype=torch.float64).scatter_add_(1, t[:2], torch.ones(2, 3, device=DEV, dtype=torch.float64))
        want = (n - 3.0 / vocab) / temperature
        # p = 2^(-log2 vocab): its argument is off by 4 u of it, so p by 4 u log2(vocab); the products and the sum by 8 u
        tol = ref.half_step(want, dtype) + ref.U * (3.0 / vocab * (4 * math.log2(vocab) + 8) + 8 * n) / temperature
        assert ref.off(dx, want, tol) <= 1


@pytest.mark.parametrize("vocab", [39, 3000])
def test_gradients_through_saved_tensors_on_the_host(vocab):
    """torch.autograd.graph.save_on_cpu, which hands dense copies of strided rows and masks back."""
    from master_doko_reinforcement_learning_amd import layer_norm, token_logprobs
    g = _gen(vocab)
    x, delta = (_randn(g, 30, vocab + 10)[:, 4:4 + vocab] for _ in range(2))
    marks = torch.rand(30, vocab + 5, generator=g, device=DEV) < 0.5
    t = torch.randint(0, vocab, (30, 2), generator=g, device=DEV)
    w = _randn(g, vocab, shift=1.0)
    for mask in (None, marks[:, 2:2 + vocab], marks[3, :vocab], marks[3, :vocab].expand(30, vocab)):
        outs = []
        for hooks in (torch.autograd.graph.save_on_cpu, torch.enable_grad):
            leaves = [u.detach().requires_grad_() for u in (x, delta, w)]
            with hooks():
                new, h = layer_norm(leaves[0], leaves[2], delta=leaves[1])
                got = token_logprobs(h, t, mask=mask)
            loss = got.logprobs.nan_to_num(neginf=0.0).sum() + got.entropy.sum() + new.sum()
            outs.append(torch.autograd.grad(loss, leaves))
        assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_vocabularies_past_32_bits_are_refused():
    from master_doko_reinforcement_learning_amd import token_logprobs
    one = torch.zeros(1, dtype=BF16, device=DEV)
    for vocab in (1 << 31, (1 << 32) + 5):
        with pytest.raises(ValueError):
            token_logprobs(one.expand(vocab))


def test_forward_mode_tangents_are_refused():
    """Neither operator has a forward derivative: a dual tensor raises, whether or not something requires a gradient."""
    from torch.autograd import forward_ad

    from master_doko_reinforcement_learning_amd import layer_norm, token_logprobs
    g = _gen(1)
    x, w, t = _randn(g, 4, 32), _randn(g, 32), torch.zeros(4, dtype=torch.int64, device=DEV)
    with forward_ad.dual_level():
        d, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        grad = _randn(g, 4, 32).requires_grad_()
        for call in (lambda: layer_norm(d), lambda: layer_norm(x, dw), lambda: layer_norm(x, None, dw), lambda: layer_norm(x, delta=d),
                     lambda: layer_norm(grad, delta=d), lambda: token_logprobs(d, t), lambda: token_logprobs(d)):
            with pytest.raises(RuntimeError):
                call()
        assert torch.equal(layer_norm(x, w), layer_norm(forward_ad.unpack_dual(d).primal, w))   # without a tangent as ever
        token_logprobs(grad, t).logprobs.sum().backward()
    assert torch.equal(layer_norm(d, dw), layer_norm(x, w))   # (the level is over, and the tangents with it)


def test_arguments_that_are_no_tensors_are_refused():
    from master_doko_reinforcement_learning_amd import layer_norm, token_logprobs
    x = torch.zeros(2, 8, device=DEV)
    for bad in (lambda: layer_norm(x, [1.0] * 8), lambda: layer_norm(x, None, 0.0), lambda: layer_norm(x, delta=[x]), lambda: token_logprobs(x, [0, 0]),
                lambda: token_logprobs(x, 0), lambda: token_logprobs(x, mask=[True] * 8)):
        with pytest.raises(ValueError):
            bad()


def test_adamw_empty_groups():
    """A group without parameters does nothing, also under a learning rate on the device."""
    from master_doko_reinforcement_learning_amd import AdamW
    lr = torch.tensor(0.5, device=DEV)
    for bits, dtype in ((32, F32), (8, BF16)):
        p = torch.zeros(3, device=DEV, dtype=dtype, requires_grad=True)
        p.grad = torch.ones_like(p)
        opt = AdamW([{"params": []}, {"params": [p]}], lr=lr, weight_decay=0.0, state_bits=bits, master_weights=True)
        opt.step()
        assert (p == -0.5).all()
        opt.load_state_dict(copy.deepcopy(opt.state_dict()))
        copy.deepcopy(opt).step()


# ------------------------------------------------------------------------------------ AdamW's masters
def _with_masters(seed, **kw):
    from master_doko_reinforcement_learning_amd import AdamW
    g = _gen(seed)
    params = [_randn(g, n, dtype=BF16, scale=0.5).requires_grad_() for n in (300, 5, 1024)]
    for p in params:
        p.grad = _randn(g, *p.shape, dtype=BF16)
    return params, AdamW(params, lr=1e-5, weight_decay=0.0, master_weights=True, **kw)   # (far below half a step of most weights)


def _same(a, b):
    (ps, o), (qs, u) = a, b
    return all(torch.equal(p, q) and torch.equal(o.state[p]["master"], u.state[q]["master"]) and torch.equal(p, o.state[p]["master"].to(p.dtype))
               for p, q in zip(ps, qs))


def _write(params, value):
    with torch.no_grad():
        for i, p in enumerate(params):
            p.copy_(torch.linspace(-value, value + i, p.numel(), device=DEV))


def test_captured_step_keeps_the_masters():
    """A step whose parameters were written to is not captured: each replay would take the rounded weights over.  After
    refresh_masters it is, and its replays are the eager steps."""
    want, mine = _with_masters(1), _with_masters(1)
    for params, opt in (want, mine):
        opt.step()
        _write(params, 0.7)                    # the weights of before a warm-up, say
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two = torch.ones(1, device=DEV) + 1
        with pytest.raises(RuntimeError, match="refresh_masters"):
            mine[1].step()
    graph.replay()
    assert float(two) == 2
    mine[1].refresh_masters()
    assert all(torch.equal(mine[1].state[p]["master"], p.float()) and int(mine[1].state[p]["step"]) == 1 for p in mine[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mine[1].step()
    for _ in range(4):
        graph.replay()
        want[1].step()
        torch.cuda.synchronize()
        assert _same(want, mine)
    assert any((mine[1].state[p]["master"] != p.float()).any() for p in mine[0])
    # what is written between replays is taken over where the caller says so
    for params, _ in (want, mine):
        _write(params, 0.3)
    mine[1].refresh_masters()
    for _ in range(3):
        graph.replay()
        want[1].step()
        torch.cuda.synchronize()
        assert _same(want, mine)


def test_raised_version_counters_leave_the_masters():
    """A parameter that holds its rounded master was not written to, whatever its version counter says (a caller raises it
    after a replay, for the networks' fused forwards)."""
    want, mine = _with_masters(2), _with_masters(2)
    for _ in range(4):
        want[1].step()
        mine[1].step()
        torch.autograd.graph.increment_version(mine[0])
        assert _same(want, mine)
    mine[1].refresh_masters()
    assert _same(want, mine)
    # a write through .data raises no counter: refresh_masters finds it
    for params, opt in (want, mine):
        for p in params:
            p.data.copy_(torch.linspace(-0.2, 0.9, p.numel(), device=DEV))
        opt.refresh_masters()
        assert all(torch.equal(opt.state[p]["master"], p.float()) for p in params)


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_follow_written_parameters(bits):
    """Parameters that were written to after the last step: a copy, a state_dict and the optimiser itself go on from the
    written values."""
    from master_doko_reinforcement_learning_amd import AdamW
    params, opt = _with_masters(3, state_bits=bits)
    opt.step()
    _write(params, 0.4)
    qs, twin = copy.deepcopy((params, opt))
    rs = [p.detach().clone().requires_grad_() for p in params]
    other = AdamW(rs, lr=1.0, weight_decay=0.0, master_weights=True, state_bits=bits)
    other.load_state_dict(opt.state_dict())
    for p, q, r in zip(params, qs, rs):
        q.grad, r.grad = p.grad.clone(), p.grad.clone()
    for _ in range(2):
        opt.step()
        twin.step()
        other.step()
        assert _same((params, opt), (qs, twin)) and _same((params, opt), (rs, other))
    assert all((opt.state[p]["master"].abs() < 3).all() and (p[-1] > 0.3) for p in params)


def test_impi_network_without_blocks():
    """forward_train without blocks is the embedding, the last LayerNorm and the head, as forward_torch."""
    from master_doko_reinforcement_learning_amd.impi_network import VOCAB_IPI, DokoImpiNet
    torch.manual_seed(0)
    net = DokoImpiNet(d=32, heads=4, layers=0).to(DEV)
    tokens = torch.cat([torch.randint(0, v, (5, 62 if i < 5 else 1)) for i, v in enumerate(VOCAB_IPI)], dim=1).int().to(DEV)
    got, want = net.forward_train(tokens), net.forward_torch(tokens)
    # one LayerNorm of sums of 6 (32 columns) and a head's products of 32: ~100 roundings of values up to ~10 times the outputs' size
    assert (got - want).abs().max() <= 100 * 10 * ref.U * want.abs().max().clamp(min=1)
    net.loss(tokens, torch.arange(5, device=DEV)).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())
