"""A training step as a program makes it: the framework's operators, the group norm over frames, backward, clip, AdamW.

A small model in the shape of a SeZM block: per-edge features from learned
matrices, attention weights (``segment_softmax``), messages summed per node
(``segment_sum``), a group norm with SiLU over the nodes of each frame, RMSNorm,
an energy per frame.  Its gradients are checked against the same model in 64
bits on the CPU, and the step against torch's clipping and AdamW in 64 bits.
"""
from __future__ import annotations

import pytest
import torch

from bysj_amd import kernels
from bysj_amd.kernels import optim
from bysj_amd.kernels.group_norm import group_norm
from parity import announce, assert_bitwise, assert_close_scaled

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FRAMES = [0, 7, 7, 20, 50]          # nodes of four frames, one of them empty
CHANNELS, GROUPS, HEADS = 24, 4, 24


def _graph(seed=0):
    generator = torch.Generator().manual_seed(seed)
    nodes = FRAMES[-1]
    degrees = torch.randint(0, 9, (nodes,), generator=generator)
    dst = torch.repeat_interleave(torch.arange(nodes), degrees)
    return {"dst": dst, "offsets": torch.cat([torch.zeros(1, dtype=torch.int64), degrees.cumsum(0)]),
            "frames": torch.tensor(FRAMES), "edges": torch.randn(dst.numel(), 16, generator=generator),
            "env": torch.rand(dst.numel(), generator=generator) + 0.1,
            "target": torch.randn(len(FRAMES) - 1, generator=generator)}


def _parameters(seed=1):
    generator = torch.Generator().manual_seed(seed)

    def draw(*shape, size=0.3):
        return torch.randn(shape, generator=generator) * size

    return {"message": draw(16, CHANNELS), "logit": draw(16, HEADS), "norm_scale": draw(CHANNELS) + 1.0,
            "norm_bias": draw(CHANNELS), "mix": draw(CHANNELS, CHANNELS), "rms_scale": draw(CHANNELS) + 1.0,
            "energy": draw(CHANNELS, 1)}


def _loss(p, g):
    """With the framework's operators, on the GPU."""
    messages = (g["edges"] @ p["message"]).contiguous()
    alpha = kernels.segment_softmax((g["edges"] @ p["logit"]).contiguous(), g["env"], g["offsets"])
    summed = kernels.segment_sum((messages * alpha).contiguous(), g["dst"], g["offsets"])
    h = group_norm(summed, GROUPS, p["norm_scale"], p["norm_bias"], offsets=g["frames"], activation="silu")
    h = kernels.rmsnorm((h @ p["mix"]).contiguous(), p["rms_scale"])
    energies = kernels.segment_sum((h @ p["energy"]).contiguous(),
                                   torch.repeat_interleave(torch.arange(len(FRAMES) - 1, device=DEV), g["frames"].diff(),
                                                           output_size=FRAMES[-1]), g["frames"])
    return (energies.squeeze(1) - g["target"]).square().sum()


def _loss_f64(p, g):
    """From the definitions, in 64 bits on the CPU."""
    nodes, dst = FRAMES[-1], g["dst"]
    edges, env = g["edges"].double(), g["env"].double()
    weighed = torch.exp(edges @ p["logit"]) * env[:, None].square()
    total = torch.zeros(nodes, HEADS, dtype=torch.float64).index_add(0, dst, weighed)
    alpha = weighed / total[dst]
    summed = torch.zeros(nodes, CHANNELS, dtype=torch.float64).index_add(0, dst, edges @ p["message"] * alpha)
    parts = []
    for a, b in zip(FRAMES, FRAMES[1:]):
        if a == b:
            continue
        rows = summed[a:b].view(b - a, GROUPS, -1)
        centred = rows - rows.mean((0, 2), keepdim=True)
        z = (centred / torch.sqrt(centred.square().mean((0, 2), keepdim=True) + 1e-5)).reshape(b - a, -1)
        z = z * p["norm_scale"] + p["norm_bias"]
        parts.append(z * torch.sigmoid(z))
    h = torch.cat(parts) @ p["mix"]
    h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * p["rms_scale"]
    per_node = (h @ p["energy"]).squeeze(1)
    energies = torch.stack([per_node[a:b].sum() for a, b in zip(FRAMES, FRAMES[1:])])
    return (energies - g["target"].double()).square().sum()


def _on_gpu(values, grad=False):
    return {k: v.to(DEV).requires_grad_(grad) for k, v in values.items()}


def test_gradients_of_the_whole_model():
    announce("training gradients")
    host, graph = _parameters(), _graph()
    p = _on_gpu(host, True)
    grads = torch.autograd.grad(_loss(p, _on_gpu(graph)), list(p.values()))
    exact = {k: v.double().requires_grad_(True) for k, v in host.items()}
    wanted = torch.autograd.grad(_loss_f64(exact, graph), list(exact.values()))
    for name, actual, expected in zip(host, grads, wanted):
        # float32 through six layers: each layer's rule is 1e-5, the frames of seven nodes amplify by 1 / std at most
        assert_close_scaled(actual, expected, rtol=1e-4, scale=1e-4, what=name)


def test_steps_follow_torch_in_64_bits():
    announce("training steps")
    host, graph = _parameters(), _graph()
    p, g = _on_gpu(host, True), _on_gpu(graph)
    optimiser = optim.AdamW(list(p.values()), lr=1e-2, weight_decay=0.05, max_norm=0.7)
    exact = {k: v.double().requires_grad_(True) for k, v in host.items()}
    theirs = torch.optim.AdamW(list(exact.values()), lr=1e-2, weight_decay=0.05, foreach=False)
    for _ in range(3):
        # the gradients are the GPU model's on both sides: the step is what is compared
        loss = _loss(p, g)
        optimiser.zero_grad()
        loss.backward()
        for k, v in exact.items():
            v.grad = p[k].grad.cpu().double()
        norm = torch.nn.utils.clip_grad_norm_(list(exact.values()), 0.7)
        optimiser.step()
        theirs.step()
        assert abs(optimiser.norm.item() / norm.item() - 1.0) < 2.0 ** -23
        for k in p:
            # ten roundings of 2^-24 a step on a step of at most 1e-2, and one on the parameter
            assert_close_scaled(p[k].detach(), exact[k].detach(), rtol=6e-7, scale=6e-7, what=k)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_training_step_replays_the_eager_one(bits):
    """Forward, backward, norm and step in one graph, replayed with eager work of a twin in between."""
    announce("captured training step", bits)
    models = []
    for _ in range(2):
        p = _on_gpu(_parameters(), True)
        models.append((p, optim.AdamW(list(p.values()), lr=1e-2, max_norm=0.7, state_bits=bits, seed=3)))
    g = _on_gpu(_graph())

    def step(p, optimiser):
        # gradients of the leaves, not accumulated into them: nothing of an earlier graph is touched
        for v, grad in zip(p.values(), torch.autograd.grad(_loss(p, g), list(p.values()))):
            v.grad = grad
        optimiser.step()
        return optimiser.norm

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(*models[0])
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(2):
        step(*models[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(*models[0])
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert_bitwise(norm, step(*models[1]), f"norm {turn}")
        for (name, a), b in zip(models[0][0].items(), models[1][0].values()):
            assert_bitwise(a.detach(), b.detach(), f"{name} {turn}")
        g["edges"].mul_(1.01)
