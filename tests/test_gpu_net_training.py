"""The networks' training path on the GPU (forward_train, loss, NetTrainer): the training operators chained as a
step uses them, against the plain modules (forward_torch, torch's autograd) in float64."""
import copy

import pytest
import torch
import torch.nn.functional as F

import net_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _exact_products():
    prev = torch.get_float32_matmul_precision()
    torch.set_float32_matmul_precision("highest")
    yield
    torch.set_float32_matmul_precision(prev)


def _impi(d=64, layers=2, batch=24, seed=0):
    from master_doko_reinforcement_learning_amd.impi_network import VOCAB_IPI, DokoImpiNet
    torch.manual_seed(seed)
    net = DokoImpiNet(d=d, heads=4, layers=layers)
    g = torch.Generator().manual_seed(seed)
    tokens = torch.cat([torch.randint(0, v, (batch, 62 if i < 5 else 1), generator=g) for i, v in enumerate(VOCAB_IPI)], dim=1).int()
    mask = torch.rand(batch, 33, generator=g) < 0.4
    guesses = torch.randint(0, 33, (batch,), generator=g)
    mask[torch.arange(batch), guesses] = True
    guesses[3] = -1
    return net, (tokens, guesses, mask)


def _az(d=64, batch=24, seed=0):
    from master_doko_reinforcement_learning_amd.az_network import VOCAB, DokoAzNet
    torch.manual_seed(seed)
    net = DokoAzNet(d=d, heads=4, layers=2)
    g = torch.Generator().manual_seed(seed)
    tokens = torch.cat([torch.randint(0, v, (batch, 62 if i < 5 else 1), generator=g) for i, v in enumerate(VOCAB)], dim=1).int()
    mask = torch.rand(batch, 39, generator=g) < 0.3
    mask[:, 5] = True
    policy = torch.rand(batch, 39, generator=g) * mask
    return net, (tokens, torch.randn(batch, 4, generator=g), policy / policy.sum(-1, keepdim=True), mask)


def _plain_loss(net, batch, entropy=0.0):
    """The same losses from forward_torch and torch's own functions."""
    if len(batch) == 3:
        tokens, guesses, mask = batch
        logits = net.forward_torch(tokens).masked_fill(~mask, -torch.inf)
        return F.cross_entropy(logits, guesses, ignore_index=-1)
    tokens, value, policy, mask = batch
    v, logits = net.forward_torch(tokens)
    lp = torch.log_softmax(logits.masked_fill(~mask, -torch.inf), -1).masked_fill(~mask, 0.0)
    ent = -(lp.exp() * lp * mask).sum(-1).mean()
    return F.mse_loss(v, value.to(v.dtype)) - (policy.to(v.dtype) * lp).sum(-1).mean() - entropy * ent


def _grads(loss, net):
    return [g.double().cpu() for g in torch.autograd.grad(loss, list(net.parameters()))]


def _distance(a, b):
    return float(torch.sqrt(sum(((x - y) ** 2).sum() for x, y in zip(a, b))))


@pytest.mark.parametrize("make", [_impi, _az])
def test_loss_and_gradients_are_as_exact_as_the_plain_modules(make):
    """Loss and all gradients against float64: no further off than twice what the plain f32 modules are (whose products
    are the same library's), plus the operators' own rounding, ~64 half steps of a gradient's norm."""
    net, batch = make()
    kw = {} if make is _impi else {"entropy": 0.01}
    exact = copy.deepcopy(net).double()
    want = _plain_loss(exact, batch, **kw)
    gw = _grads(want, exact)
    net, batch = net.to(DEV), tuple(t.to(DEV) for t in batch)
    plain = _plain_loss(net, batch, **kw)
    gp = _grads(plain, net)
    got = net.loss(*batch, **kw)
    gg = _grads(got, net)
    size = _distance(gw, [torch.zeros_like(g) for g in gw])
    assert _distance(gg, gw) <= 2 * _distance(gp, gw) + 64 * ref.U * size
    got, plain, want = got.item(), plain.item(), want.item()
    assert abs(got - want) <= 2 * abs(plain - want) + 64 * ref.U * abs(want)
    # the forwards agree as closely
    with torch.no_grad():
        a, b = net.forward_train(batch[0]), net.forward_torch(batch[0])
        for x, y in zip((a, ) if torch.is_tensor(a) else a, (b, ) if torch.is_tensor(b) else b):
            # 2 blocks of ~10 roundings over sums of 256 products, of values up to ~10 times the output's scale
            assert (x - y).abs().max() <= 20 * 256 * 10 * ref.U * y.abs().max().clamp(min=1)


@pytest.mark.parametrize("make,bits", [(_impi, 32), (_impi, 8), (_az, 32)])
def test_trainer_steps(make, bits):
    """Three steps: each parameter moves as AdamW's formula says for the gradients that the step took."""
    from master_doko_reinforcement_learning_amd import NetTrainer
    net, batch = make(d=32)
    net, batch = net.to(DEV), tuple(t.to(DEV) for t in batch)
    hyper = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.01)
    trainer = NetTrainer(net, state_bits=bits, **hyper)
    state = trainer.optimizer.state
    for t in range(1, 4):
        before = []
        for p in net.parameters():
            st = state[p]
            m, v = st["exp_avg"].float().double().reshape(-1), st["exp_avg_sq"].float().double().reshape(-1)
            if bits == 8:
                n = p.numel()
                m = m * st["exp_avg_scale"].double().repeat_interleave(256)[:n]
                v = (v * st["exp_avg_sq_scale"].double().repeat_interleave(256)[:n]) ** 2
            before.append((p.detach().double().reshape(-1), m, v))
        loss = trainer.step(*batch)
        assert loss.shape == () and torch.isfinite(loss) and not loss.requires_grad
        for p, (w, m, v) in zip(net.parameters(), before):
            (p1, _, _), (tp, _, _) = ref.adamw(w, p.grad.double().reshape(-1), m, v, t, hyper["lr"], hyper["betas"], hyper["eps"], hyper["weight_decay"])
            assert ref.off(p.detach().reshape(-1), p1, tp) <= 1


@pytest.mark.parametrize("make,d", [(_impi, 256), (_az, 160)])
def test_fused_inference_follows_a_training_step(make, d):
    """The fused forwards keep split and folded weights: after a step they are those of the new parameters."""
    from master_doko_reinforcement_learning_amd import NetTrainer
    net, batch = make(d=d, batch=8)
    net, batch = net.to(DEV), tuple(t.to(DEV) for t in batch)
    first = lambda o: o if torch.is_tensor(o) else o[1]  # noqa: E731
    with torch.no_grad():
        old = first(net(batch[0]))
    trainer = NetTrainer(net, lr=3e-3)
    for _ in range(2):
        trainer.step(*batch)
    with torch.no_grad():
        new, want = first(net(batch[0])), first(net.forward_torch(batch[0]))
    # bf16x3 products of ~16 bits against a change of the weights by 2 x 3e-3
    assert (new - want).abs().max() <= 2e-3 * want.abs().max() and (new - old).abs().max() > 2e-2 * want.abs().max()


def test_trainer_state_round_trip():
    from master_doko_reinforcement_learning_amd import NetTrainer
    net, batch = _impi(d=32)
    net, batch = net.to(DEV), tuple(t.to(DEV) for t in batch)
    a = NetTrainer(net, lr=1e-3, state_bits=8)
    a.step(*batch)
    twin, _ = _impi(d=32, seed=5)
    b = NetTrainer(twin.to(DEV), lr=1.0, state_bits=8)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    # (the embeddings' gradients are summed by atomics, so the two runs' gradients may differ in their last bits: give both the same)
    for p, q in zip(net.parameters(), b.net.parameters()):
        assert torch.equal(p, q)
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    a.optimizer.step()
    b.optimizer.step()
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), b.net.parameters()))


def test_impi_logprobs_of_guesses():
    """DokoImpiNet.logprobs against log_softmax in float64 of the same logits: the sampler's distribution."""
    net, (tokens, guesses, mask) = _impi(d=256, batch=16)
    net, tokens, guesses, mask = net.to(DEV), tokens.to(DEV), guesses.to(DEV), mask.to(DEV)
    with torch.no_grad():
        logits = net(tokens)
    got = net.logprobs(tokens, guesses, mask=mask, temperature=0.8, top=3)
    want, lp, _ = ref.logp(logits.double(), guesses[:, None], mask, 0.8)
    assert ref.off(got.logprobs[:, None], *want["logprobs"]) <= 1 and ref.off(got.entropy, *want["entropy"]) <= 1
    assert torch.equal(got.top_tokens, torch.sort(torch.where(mask, logits, -torch.inf), dim=-1, descending=True, stable=True).indices[:, :3])


def test_trainer_refuses():
    from master_doko_reinforcement_learning_amd import NetTrainer
    net, _ = _impi(d=32)
    with pytest.raises(ValueError):
        NetTrainer(net)
    with pytest.raises(ValueError):
        NetTrainer(net.to(DEV).bfloat16())
    net, batch = _impi(d=32)
    trainer, batch = NetTrainer(net.to(DEV)), tuple(t.to(DEV) for t in batch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two = torch.ones(1, device=DEV) + 1
        with pytest.raises(RuntimeError):
            trainer.step(*batch)
    graph.replay()
    assert float(two) == 2
    trainer.step(*batch)
