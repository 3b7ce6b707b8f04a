"""The decoder of feature rows and the rendering path that runs it: the index map's rows through products, norms and
dropout to an image, and back to the Gaussians' feature vectors and the decoder's weights."""
import math

import pytest
import torch

import decoder_reference as ref
from neuralgaussiansplatting_amd import synthetic
from neuralgaussiansplatting_amd.cameras import make_camera
from neuralgaussiansplatting_amd.feature_decoder import FeatureDecoder

DEV = "cuda:0"


def test_parameters_and_refusals():
    d = FeatureDecoder(width=96, blocks=3)
    assert sum(p.numel() for p in d.parameters()) == 64 * 96 + 96 + 3 * (2 * 96 + 2 * (96 * 96 + 96)) + 2 * 96 + 96 * 3 + 3
    again = FeatureDecoder(width=96, blocks=3)
    again.load_state_dict(d.state_dict())
    with pytest.raises(ValueError):
        FeatureDecoder(dropout=1.5)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        d(torch.zeros(4, 64))


def in_double(decoder, x, seed, training):
    """The decoder's formula on torch's operators in 64 bits, on copies of its parameters."""
    p = {n: t.detach().double().requires_grad_() for n, t in decoder.named_parameters()}
    x = x.detach().double().requires_grad_()
    f = torch.nn.functional
    lin = lambda t, n: t @ p[n + ".weight"].t() + p[n + ".bias"]
    norm = lambda t, n: f.layer_norm(t, t.shape[-1:], p[n + ".weight"], p[n + ".bias"], 1e-5)
    h = f.gelu(lin(x, "lift"))
    for i in range(len(decoder.ups)):
        t = lin(f.gelu(lin(norm(h, "norms.%d" % i), "ups.%d" % i)), "downs.%d" % i)
        if training:
            drop = round(decoder.dropout * 65536)
            mask = ref.kept(t.numel(), decoder.dropout, seed, i).view(t.shape).to(t.device)
            t = torch.where(mask, t * (65536 / (65536 - drop)), 0.0)
        h = h + t
    return torch.sigmoid(lin(norm(h, "head_norm"), "head")), x, p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,training", [(1, False), (130, True), (4608, True), (4608, False)])
def test_decoder_against_torch(rows, training, dtype):
    """Values and gradients against 64 bits.  On the way there each of at most 9 operators rounds once (float32: sums of
    at most 128 terms, 130 e), on the way back each product rounds its dz and its result; no step amplifies a relative
    error by more than 4 in norm (see test_decoder_ops_gpu.test_block): 9 + 18 roundings times 4.  A gradient's sums over
    the rows add rows times e."""
    torch.manual_seed(7)
    d = FeatureDecoder(dropout=0.2, device=DEV, dtype=dtype).train(training)
    x = torch.randn(rows, 64, device=DEV).to(dtype).requires_grad_()
    dy = torch.randn(rows, 3, device=DEV).to(dtype)
    y = d(x, 5)
    names = [n for n, _ in d.named_parameters()]
    grads = torch.autograd.grad(y, [x] + list(d.parameters()), dy)
    want, x64, p64 = in_double(d, x, 5, training)
    want_grads = torch.autograd.grad(want, [x64] + [p64[n] for n in names], dy.double())
    bar = 4 * 27 * (ref.half_step(dtype) if dtype != torch.float32 else (130 + rows) * ref.E)
    assert (y.double() - want).norm() <= bar * want.norm()
    for n, got, w in zip(["x"] + names, grads, want_grads):
        assert (got.double() - w).norm() <= bar * w.norm(), n


class Model:
    """The read interface render_features asks of a Gaussian model."""
    active_sh_degree = 0

    def __init__(self, means, features):
        self.get_xyz, self._features = means, features


@pytest.mark.gpu
def test_render_features():
    from neuralgaussiansplatting_amd.gaussian_renderer import PipelineParams, render_features
    W, H, P = 100, 76, 3000
    sc = synthetic.make_scene(P, 0, (-3.0, -2.0), seed=3)
    cam = make_camera(W, H, synthetic.FOVX, (0.5, 0.4, -4.0), device=torch.device(DEV))
    torch.manual_seed(3)
    pc = Model(sc.means3D.to(DEV).requires_grad_(), torch.randn(P, 64, device=DEV, requires_grad=True))
    d = FeatureDecoder(width=64, blocks=1, dropout=0.1, device=DEV)
    bg = torch.tensor([0.25, 0.5, 0.75], device=DEV)
    out = render_features(cam, pc, d, PipelineParams(), bg, seed=11)
    image, hit = out["render"], out["idxmap"] >= 0
    assert image.shape == (3, H, W) and hit.any() and not hit.all()
    assert (image[:, ~hit].t() == bg).all()
    # the image is the decoder's on the feature map, and the gradients arrive where they belong
    want, rows64, p64 = in_double(d, out["feature_map"], 11, True)
    image64 = torch.where(hit.unsqueeze(-1), want, bg.double()).permute(2, 0, 1)
    bar = 4 * 27 * (130 + H * W) * ref.E
    assert (image.double() - image64).norm() <= bar * image64.norm()
    dL = torch.randn(3, H, W, device=DEV)
    names = [n for n, _ in d.named_parameters()]
    grads = torch.autograd.grad(image, [pc._features] + list(d.parameters()), dL)
    want_grads = torch.autograd.grad(image64, [rows64] + [p64[n] for n in names], dL.double())
    per_gaussian = torch.zeros(P, 64, device=DEV, dtype=torch.float64)
    per_gaussian.index_add_(0, out["idxmap"][hit].long(), want_grads[0][hit])
    per_gaussian[:, :25] = 0  # depth and direction take their places in the row
    for n, got, w in zip(["features"] + names, grads, (per_gaussian,) + want_grads[1:]):
        assert (got.double() - w).norm() <= bar * w.norm(), n
    # another seed, another mask; none outside training
    assert not torch.equal(render_features(cam, pc, d, PipelineParams(), bg, seed=12)["render"], image)
    d.eval()
    a, b = (render_features(cam, pc, d, PipelineParams(), bg, seed=s)["render"] for s in (1, 2))
    assert torch.equal(a, b)
    # a decoder in bfloat16 reads the map in its type and gives an image in the map's
    half = FeatureDecoder(width=64, blocks=1, device=DEV, dtype=torch.bfloat16).eval()
    half.load_state_dict(d.state_dict())
    c = render_features(cam, pc, half, PipelineParams(), bg)["render"]
    assert c.dtype == torch.float32 and (c - a).norm() <= 4 * 27 * ref.half_step(torch.bfloat16) * a.norm()
