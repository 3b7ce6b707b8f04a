"""What render_features hands to the decoder and makes of its answer, with the index map's rasterizer replaced."""
import types

import torch

from neuralgaussiansplatting_amd import gaussian_renderer as gr

H, W = 3, 4


def test_the_decoder_may_be_any_callable(monkeypatch):
    """The decoder is a map from feature rows and a seed to colours; it need not be a module."""
    rows = torch.arange(H * W * 64, dtype=torch.float32).view(H, W, 64)
    hit = torch.tensor([[0, -1, 2, 3], [-1, 5, 6, 7], [8, 9, -1, 11]], dtype=torch.int32)

    class Rasterizer:
        def __init__(self, raster_settings):
            pass

        def __call__(self, *_):
            return hit, None, torch.ones(H, W), rows

    monkeypatch.setattr(gr, "GaussianRasterizer2", Rasterizer)
    cam = types.SimpleNamespace(image_height=H, image_width=W, FoVx=1.0, FoVy=1.0, world_view_transform=torch.eye(4),
                                full_proj_transform=torch.eye(4), camera_center=torch.zeros(3))
    pc = types.SimpleNamespace(active_sh_degree=0, get_xyz=torch.zeros(12, 3), _features=torch.zeros(12, 64))
    bg = torch.tensor([0.25, 0.5, 0.75])
    seen = []

    def decoder(features, seed):
        seen.append((features.dtype, seed))
        return features[..., :3] * 2

    out = gr.render_features(cam, pc, decoder, gr.PipelineParams(), bg, seed=9)
    assert seen == [(torch.float32, 9)]
    want = torch.where((hit >= 0).unsqueeze(-1), rows[..., :3] * 2, bg)
    assert torch.equal(out["render"], want.permute(2, 0, 1))
