"""A scene over frames, trained as a user would: projections of per-Gaussian
features give the gates and inputs of gated_scan, its states move the Gaussians
of each frame, render() and fused_ssim give the loss, and the projections are
updated by muon_step, the Gaussians by the trainer's Adam."""
import importlib

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"
N, FRAMES, FEATURES, W, H = 400, 5, 12, 64, 48


def plain_scan(x, g):
    """The recurrence row by row, in autograd's own operations."""
    h, rows = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        h = g[:, t] * h + x[:, t]
        rows.append(h)
    return torch.stack(rows, 1), h


def scene(gs):
    cfg = gs.scenes.CONFIGS[0]
    raw = {k: v.to(DEV).clone().requires_grad_(True) for k, v in gs.scenes.make_gaussians(cfg, seed=5, n=N).items()}
    gen = torch.Generator(device=DEV).manual_seed(6)
    z = torch.randn(N, FRAMES, FEATURES, generator=gen, device=DEV)
    wx = (0.02 * torch.randn(FEATURES, 3, generator=gen, device=DEV)).requires_grad_(True)
    wg = (0.3 * torch.randn(FEATURES, 3, generator=gen, device=DEV)).requires_grad_(True)
    target = 255 * torch.rand(FRAMES, H, W, 3, generator=gen, device=DEV)
    w2c = gs.scenes.primary_camera(cfg).to(DEV)
    K = torch.tensor([[80.0, 0, W / 2], [0, 80.0, H / 2], [0, 0, 1]], device=DEV)
    return raw, z, wx, wg, target, w2c, K


def loss_of(gs, scan, raw, z, wx, wg, target, w2c, K):
    ssim = importlib.import_module("3dgs_from_scratch_b200.ssim").fused_ssim
    h, final = scan(z @ wx, torch.sigmoid(z @ wg))
    act = gs.scenes.activate(raw)
    total = 1e-3 * final.square().sum()
    for t in range(FRAMES):
        img, _, _ = gs.render(w2c, K, W, H, act["means"] + h[:, t], act["scales"], act["quaternions"],
                              act["opacities"], act["sh_coeffs_dc"], act["sh_coeffs_rest"])
        a, b = (v.permute(2, 0, 1)[None] / 255 for v in (img, target[t]))
        total = total + 0.8 * (a - b).abs().mean() + 0.2 * (1 - ssim(a, b, padding="valid"))
    return total


@gpu
def test_a_training_step_through_the_recurrence(gs):
    s = scene(gs)
    raw, wx, wg = s[0], s[2], s[3]
    leaves = [wx, wg] + list(raw.values())
    got = torch.autograd.grad(loss_of(gs, gs.gated_scan, *s), leaves)
    ref = torch.autograd.grad(loss_of(gs, plain_scan, *s), leaves)
    for name, a, b in zip(["wx", "wg"] + list(raw), got, ref):
        # the same images but for fp32 rounding; the rasterizer's own gradients carry
        # atomics whose order changes between runs
        assert bool(torch.isfinite(a).all()), name
        assert float((a - b).norm()) <= 1e-3 * float(b.norm()) + 1e-12, name
    assert float(got[0].norm()) > 0 and float(got[1].norm()) > 0

    dp = importlib.import_module("3dgs_from_scratch_b200.dp")
    fp = dp.FlatParams({k: v.detach().clone() for k, v in raw.items()})
    before = fp.data.clone()
    for p, grad in zip(fp.params.values(), got[2:]):
        p.grad.copy_(grad)
    fp.step()
    weights = [w.detach().clone() for w in (wx, wg)]
    momentum = [torch.zeros_like(w) for w in weights]
    for w, m, grad in zip(weights, momentum, got[:2]):
        old = w.clone()
        gs.muon_step(w, grad, m, 0.02)
        step = (old - w).double().cpu()
        # 12 x 3: scale 2; singular values of the update end in the quintic's band
        values = torch.linalg.svdvals(step) / (0.02 * 2)
        assert float(values.max()) < 1.21 and bool(torch.isfinite(w).all())
        assert torch.allclose(m, 0.05 * grad, rtol=1e-6, atol=0)
    assert not torch.equal(before, fp.data) and bool(torch.isfinite(fp.data).all())


@gpu
def test_frame_by_frame_gives_the_trained_states(gs):
    raw, z, wx, wg = scene(gs)[:4]
    with torch.no_grad():
        x, g = z @ wx, torch.sigmoid(z @ wg)
        h, final = gs.gated_scan(x, g)
        state = torch.zeros(N, 3, device=DEV)
        for t in range(FRAMES):
            row, state = gs.gated_scan(x[:, t:t + 1], g[:, t:t + 1], initial=state)
            assert torch.allclose(row[:, 0], h[:, t], rtol=0, atol=20 * 2.0 ** -24)
        assert torch.allclose(state, final, rtol=0, atol=20 * 2.0 ** -24)
