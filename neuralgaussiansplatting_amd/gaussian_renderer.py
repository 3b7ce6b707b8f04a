"""Caller-side counterpart of the reference's ``render()``
(gaussian_renderer/__init__.py:19-101): builds the raster settings from a
camera and a Gaussian model, chooses the SH / covariance code paths from the
pipeline flags, calls the rasterizer and packages the result dict.

``pc`` is any object with the reference model's read interface
(scene/gaussian_model.py:113-144): ``get_xyz, get_opacity, get_scaling,
get_rotation, get_features, get_covariance(scaling_modifier),
active_sh_degree, max_sh_degree``.  ``pipe`` carries ``debug``,
``compute_cov3D_python`` and ``convert_SHs_python``
(arguments/__init__.py:64-69).
"""
import math

import torch

from .diff_gaussian_rasterization import GaussianRasterizationSettings, GaussianRasterizer
from .rasterizer2 import GaussianRasterizationSettings2, GaussianRasterizer2
from .sh_utils import eval_sh


class PipelineParams:
    """Defaults of the reference's pipeline flag group (arguments/__init__.py:64-69)."""

    def __init__(self, convert_SHs_python=False, compute_cov3D_python=False, debug=False):
        self.convert_SHs_python = convert_SHs_python
        self.compute_cov3D_python = compute_cov3D_python
        self.debug = debug


def render(viewpoint_camera, pc, pipe, bg_color, scaling_modifier=1.0, override_color=None):
    """Render the scene.  ``bg_color`` must live on the GPU.  Returns
    ``{"render", "viewspace_points", "visibility_filter", "radii"}``."""
    xyz = pc.get_xyz
    # zero tensor whose gradient receives dL/d(screen-space mean); densification reads it
    screenspace_points = torch.zeros_like(xyz, dtype=xyz.dtype, requires_grad=True, device=xyz.device) + 0
    try:
        screenspace_points.retain_grad()
    except Exception:
        pass

    settings = GaussianRasterizationSettings(
        image_height=int(viewpoint_camera.image_height),
        image_width=int(viewpoint_camera.image_width),
        tanfovx=math.tan(viewpoint_camera.FoVx * 0.5),
        tanfovy=math.tan(viewpoint_camera.FoVy * 0.5),
        bg=bg_color,
        scale_modifier=scaling_modifier,
        viewmatrix=viewpoint_camera.world_view_transform,
        projmatrix=viewpoint_camera.full_proj_transform,
        sh_degree=pc.active_sh_degree,
        campos=viewpoint_camera.camera_center,
        prefiltered=False,
        debug=pipe.debug,
    )
    rasterizer = GaussianRasterizer(raster_settings=settings)

    scales = rotations = cov3D_precomp = None
    if pipe.compute_cov3D_python:
        cov3D_precomp = pc.get_covariance(scaling_modifier)
    else:
        scales, rotations = pc.get_scaling, pc.get_rotation

    shs = colors_precomp = None
    if override_color is not None:
        colors_precomp = override_color
    elif pipe.convert_SHs_python:
        feats = pc.get_features
        shs_view = feats.transpose(1, 2).view(-1, 3, (pc.max_sh_degree + 1) ** 2)
        dir_pp = xyz - viewpoint_camera.camera_center.repeat(feats.shape[0], 1)
        dir_pp = dir_pp / dir_pp.norm(dim=1, keepdim=True)
        colors_precomp = torch.clamp_min(eval_sh(pc.active_sh_degree, shs_view, dir_pp) + 0.5, 0.0)
    else:
        shs = pc.get_features

    rendered_image, radii = rasterizer(means3D=xyz, means2D=screenspace_points, shs=shs,
                                       colors_precomp=colors_precomp, opacities=pc.get_opacity, scales=scales,
                                       rotations=rotations, cov3D_precomp=cov3D_precomp)
    return {"render": rendered_image, "viewspace_points": screenspace_points, "visibility_filter": radii > 0,
            "radii": radii}


def render_features(viewpoint_camera, pc, decoder, pipe, bg_color, seed=0):
    """Render through the index map and a decoder: every pixel's feature row (depth, encoded view direction, features
    25..63 of the nearest Gaussian) is decoded to a colour; pixels that show no Gaussian get ``bg_color``.  The per-pixel
    counterpart of the reference's neural front-end (gaussian_renderer/__init__.py:104-210).  ``pc`` also carries the
    feature vectors ``_features`` [P, 64] (scene/gaussian_model.py:176), which receive gradients; ``decoder`` maps
    [H, W, 64] and a dropout seed to [H, W, 3], e.g. a ``FeatureDecoder``.  Returns
    ``{"render" [3, H, W], "idxmap", "depth", "feature_map"}``."""
    settings = GaussianRasterizationSettings2(
        image_height=int(viewpoint_camera.image_height),
        image_width=int(viewpoint_camera.image_width),
        tanfovx=math.tan(viewpoint_camera.FoVx * 0.5),
        tanfovy=math.tan(viewpoint_camera.FoVy * 0.5),
        bg=bg_color,
        scale_modifier=1.0,
        viewmatrix=viewpoint_camera.world_view_transform,
        projmatrix=viewpoint_camera.full_proj_transform,
        sh_degree=pc.active_sh_degree,
        campos=viewpoint_camera.camera_center,
        prefiltered=False,
        debug=pipe.debug,
    )
    # (the index map takes its place from the centres alone and has gradients for the feature vectors alone)
    xyz = pc.get_xyz.detach()
    idxmap, _, depth, feature_map = GaussianRasterizer2(raster_settings=settings)(xyz, None, xyz, pc._features)
    # (a decoder with weights gets the rows in their type, any other callable as they are)
    weights = getattr(decoder, "parameters", tuple)()
    dtype = next((p.dtype for p in weights), feature_map.dtype)
    colors = decoder(feature_map.to(dtype), seed).to(feature_map.dtype)
    image = torch.where((idxmap >= 0).unsqueeze(-1), colors, bg_color.to(colors.dtype))
    return {"render": image.permute(2, 0, 1), "idxmap": idxmap, "depth": depth, "feature_map": feature_map}
