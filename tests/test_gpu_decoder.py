"""The decoder operators together, as they are used: Gaussians blend custom features into a feature image, two
normalised layers decode it to colour, GaussianMuon steps the layers' matrices and GaussianAdam the rest."""
import pytest
import torch
from torch.nn import functional as F

import d3gs_research_b200 as d3
from d3gs_research_b200 import GaussianAdam, GaussianMuon, group_norm_act
from d3gs_research_b200.config_def import EarlyFilterAlgo
from parity_utils import gpu_cameras, gpu_model, small_scene

pytestmark = pytest.mark.gpu


def test_feature_image_decoded_and_trained(cuda_device):
    sc = small_scene(n=2048, width=96, height=64, sh_degree=3, seed=6)
    op = d3.GaussianSplatOp(d3.GaussianSplatConfig(early_filter_algo=EarlyFilterAlgo.OBB_DFVT))
    model, cams = gpu_model(sc, cuda_device), gpu_cameras(sc, cuda_device)
    model.act_applied = True
    g = torch.Generator(device="cuda").manual_seed(0)
    features = torch.randn(2048, 12, generator=g, device="cuda").requires_grad_()
    mats = [torch.nn.Parameter(torch.randn(o, i, generator=g, device="cuda") / i ** 0.5) for o, i in ((24, 12), (24, 24), (3, 24))]
    norms = [torch.nn.Parameter(t) for t in (torch.ones(24, device="cuda"), torch.zeros(24, device="cuda"),
                                             torch.ones(24, device="cuda"), torch.zeros(24, device="cuda"))]
    target = torch.rand(1, 64, 96, 3, generator=g, device="cuda")
    muon = GaussianMuon(mats, lr=0.02, weight_decay=0.0)
    adam = GaussianAdam([{"params": norms}, {"params": [features]}], lr=1e-2, eps=1e-15)

    def decode(image, norm):
        h = norm(image @ mats[0].T, norms[0], norms[1])
        h = norm(h @ mats[1].T, norms[2], norms[3])
        return torch.sigmoid(h @ mats[2].T)

    own = lambda h, w, b: group_norm_act(h, 4, w, b)   # noqa: E731
    plain = lambda h, w, b: F.silu(F.group_norm(h.permute(0, 3, 1, 2), 4, w, b)).permute(0, 2, 3, 1)   # noqa: E731
    leaves = [features, *mats, *norms]
    for step in range(2):
        out = d3.rasterize_gaussians(model, cams, op=op, training=True, custom_features=features)
        image = out.custom_features
        assert image.shape == (1, 64, 96, 12)
        want = torch.autograd.grad(F.mse_loss(decode(image, plain), target), leaves, retain_graph=True)
        for t in leaves:
            t.grad = None
        F.mse_loss(decode(image, own), target).backward()
        for t, w in zip(leaves, want):
            # both sides differ from the formula by 32-bit rounding in sums over 6144 pixels and three layers
            assert torch.linalg.vector_norm(t.grad - w) <= 1e-4 * torch.linalg.vector_norm(w)
        before = [t.detach().clone() for t in leaves]
        muon.step()
        adam.step()
        for t, b in zip(leaves, before):
            assert torch.isfinite(t).all() and not torch.equal(t, b)
        for m, b in zip(mats, before[1:4]):
            # singular values of the step lie around lr * sqrt(max(1, rows / columns)), within the polynomial's band
            s = torch.linalg.svdvals((b - m).detach()) / (0.02 * max(1.0, m.shape[0] / m.shape[1]) ** 0.5)
            assert s.max() < 1.25
