"""The appearance head on a frozen cloud: its gradients against torch's own in 64 bits, and a short training with moments in
32 and in 8 bits."""
import math

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

import numpy as np

pytestmark = pytest.mark.gpu


def plain(head, features, image):
    """The head in 64 bits on the CPU, from copies of its parameters."""
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in head.named_parameters()}

    def norm(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    x = norm(features.cpu().double(), p["norm_weight"], p["norm_bias"])
    stream = x @ p["enter.weight"].t() + p["enter.bias"] + p["embedding"][image] @ p["mix.weight"].t()
    for i in range(len(head.blocks)):
        b = f"blocks.{i}."
        u = norm(stream, p[b + "norm_weight"], p[b + "norm_bias"]) @ p[b + "up.weight"].t() + p[b + "up.bias"]
        stream = stream + torch.nn.functional.gelu(u) @ p[b + "down.weight"].t() + p[b + "down.bias"]
    return norm(stream, p["last_weight"], p["last_bias"]) @ p["leave.weight"].t() + p["leave.bias"], p


def test_gradients_against_64_bits():
    import appearance_head
    import splatx_torch
    b = splatx_torch.TorchBackend(0)
    torch.manual_seed(3)
    head = appearance_head.AppearanceHead(b, 12, 3, hidden=20, embedding=5, dtype=torch.float32)
    torch.nn.init.normal_(head.leave.weight)
    features, c = torch.randn(777, 12, device="cuda"), torch.randn(777, 3, device="cuda")
    out = head(features, 1)
    (out * c).sum().backward()
    want, p = plain(head, features, 1)
    (want * c.cpu().double()).sum().backward()
    # a dozen operations of 32 bits with sums of at most 777 terms: some thousands of units of 2^-24 of the largest value
    assert (out.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()
    for k, v in head.named_parameters():
        g = p[k].grad
        assert (v.grad.cpu().double() - g).norm() <= 1e-4 * g.norm() + 1e-12, k
    b.close()


@pytest.mark.parametrize("state_bits", [32, 8])
def test_training_follows_the_images(state_bits):
    import appearance_head
    losses = appearance_head.demo(n=3000, images=3, steps=90, state_bits=state_bits, width=96, height=64, sh_degree=2, quiet=True)
    assert all(math.isfinite(x) for x in losses)
    assert np.mean(losses[-6:]) < 0.5 * np.mean(losses[:3])
