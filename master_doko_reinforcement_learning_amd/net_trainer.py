"""A training step of the networks on the GPU: the counterpart of AzEvaluator on the learning side (the
reference's NetworkWithTrainer.fit, rs-doko-py-bridge/python/az_doko.py)."""
import torch

from .net_ops import AdamW


class NetTrainer:
    """Fits a DokoAzNet or DokoImpiNet (f32, on the GPU) with AdamW: step(*batch) is one pass of net.loss(*batch),
    its gradients (net_ops.layer_norm, net_ops.token_logprobs) and the update of every parameter.

    state_bits 8 keeps the optimiser's moments in 8 bits.  The networks' fused forwards notice new weights by
    themselves, so an AzEvaluator or ARSampling on the same net goes on with what was learnt."""

    def __init__(self, net, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        params = list(net.parameters())
        if any(p.dtype != torch.float32 or not p.is_cuda for p in params):
            raise ValueError("NetTrainer: the network is trained in float32 on the GPU")
        self.net = net
        self.optimizer = AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits)

    def step(self, *batch, **kwargs):
        """One step on net.loss(*batch, **kwargs); returns the loss before it (on the device, not synchronised).
        Not to be captured into a graph: the library calls of the networks' heads and embeddings are not."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("NetTrainer.step is not captured into graphs (AdamW.step is)")
        self.optimizer.zero_grad(set_to_none=True)
        # (the backward pass on this thread, not on the engine's for the GPU: without the hand-over of every step a
        # batch of 64 positions takes 4.1 ms instead of 4.7, IMPI network)
        with torch.enable_grad(), torch.autograd.set_multithreading_enabled(False):
            loss = self.net.loss(*batch, **kwargs)
            loss.backward()
        self.optimizer.step()
        return loss.detach()

    def state_dict(self):
        return {"net": self.net.state_dict(), "optimizer": self.optimizer.state_dict()}

    def load_state_dict(self, state_dict):
        self.net.load_state_dict(state_dict["net"])
        self.optimizer.load_state_dict(state_dict["optimizer"])
