"""Plane statistics through the cost-volume managers, the models (eager, captured graphs, launch programs) and the fusing loops."""
import numpy as np
import pytest
import torch

import plane_ref as ref
from doubletake_amd.modules import plane_ops
from doubletake_amd.utils import synthetic as syn

pytestmark = pytest.mark.gpu
KEYS = ("plane_log_prob_bhw", "plane_entropy_bhw", "plane_top_log_prob_bkhw", "plane_top_depth_bkhw")


def _model(kind="hint", h=24, w=32, k=3, D=16, b=2, dec="skip", seed=5):
    import gpu_util as gu
    from doubletake_amd.experiment_modules.doubletake_model import DepthModel, DepthModelCVHint

    enc, widths = ("resnet18d", [64, 64, 128, 256, 512]) if dec == "skip" else ("efficientnet", [24, 48, 64, 160, 256])
    kw = dict(image_encoder_name=enc, depth_decoder_name=dec, matching_num_depth_bins=D, model_num_views=k + 1, matching_encoder_type=None)
    model = DepthModelCVHint(4 * h, 4 * w, **kw) if kind == "hint" else DepthModel(4 * h, 4 * w, feature_volume_type=kind, **kw)
    gu.set_formula_weights(model, seed)
    model = model.to(gu.dev())

    def frame(s):
        t = gu.to_dev(syn.volume_inputs(b, k, h, w, 16, s))
        pyr = [torch.from_numpy(p).to(gu.dev()).contiguous(memory_format=torch.channels_last)
               for p in syn.prior_pyramid(b, widths, 2 * h, 2 * w, s + 50)]
        return t, pyr

    def run(fr):
        t, pyr = fr
        return model.forward_from_features(pyr, t["cur_feats"], t["src_feats"], t["src_extrinsics"], t["src_poses"], t["src_Ks"],
                                           t["cur_invK"], gu.hint_dict(t) if kind == "hint" else None, return_mask=True)

    def volume(fr):
        kw = gu.volume_call_args(fr[0])
        kw["min_depth"] = torch.full((1, 1, 1, 1), model.min_matching_depth, device=gu.dev())
        kw["max_depth"] = torch.full((1, 1, 1, 1), model.max_matching_depth, device=gu.dev())
        if kind == "hint":
            kw["cv_depth_hint_dict"] = gu.hint_dict(fr[0])
        return model.cost_volume(**kw)

    return model, frame, run, volume


@pytest.mark.parametrize("kind,dec", [("hint", "skip"), ("hint", "unet_pp"), ("mlp_feature_volume", "skip"), ("simple_cost_volume", "skip")])
def test_model_outputs_against_the_64_bit_form(kind, dec):
    model, frame, run, volume = _model(kind, dec=dec)
    fr = frame(11)
    before = {k: v.clone() for k, v in run(fr).items() if isinstance(v, torch.Tensor)}
    assert not any(k in before for k in KEYS)
    model.enable_plane_statistics(top=3, scale=2.0)
    out = run(fr)
    for k, v in before.items():   # what ran before keeps its results
        assert torch.equal(out[k], v), k
    vol, low, planes, _ = volume(fr)
    depth = out["depth_pred_s1_b1hw"]
    assert depth.shape[-2:] == vol.shape[-2:]
    idx = ref.nearest(depth[:, 0], planes)
    want = ref.stats(vol, idx, 3, 2.0, None, planes)
    D = vol.shape[1]
    ref.close(out[KEYS[0]], want["log_prob"], ref.bound_a(D), 4 * ref.U, "log_prob")
    ref.close(out[KEYS[1]], want["entropy"], ref.bound_b(D), 0.0, "entropy")
    ref.close(out[KEYS[2]], want["top_log_prob"], ref.bound_a(D), 4 * ref.U, "top")
    assert torch.equal(out[KEYS[3]].cpu(), want["top_depth"])
    assert torch.equal(out[KEYS[3]][:, 0], low) and torch.equal(low, out["lowest_cost_bhw"])   # the most probable plane is the argmax
    model.enable_plane_statistics(top=0)
    out = run(fr)
    assert KEYS[0] in out and KEYS[2] not in out
    model.enable_plane_statistics(False)
    assert not any(k in run(fr) for k in KEYS)


@pytest.mark.parametrize("how", ["graphs", "programs"])
def test_replays_equal_eager_and_follow_the_setting(how):
    model, frame, run, _ = _model(b=1)
    model.enable_plane_statistics(top=2)
    frames = [frame(s) for s in (1, 2, 3)]
    want = [{k: v.clone() for k, v in run(f).items() if isinstance(v, torch.Tensor)} for f in frames]
    (model.enable_hip_graphs if how == "graphs" else model.enable_launch_programs)(True)
    for _ in range(2):
        for f, ww in zip(frames, want):
            out = run(f)
            torch.cuda.synchronize()
            for k in ww:
                assert torch.equal(out[k], ww[k]), k
    model.enable_plane_statistics(False)
    assert not any(k in run(frames[0]) for k in KEYS)
    model.enable_plane_statistics(top=2, scale=0.5)
    out = {k: v.clone() for k, v in run(frames[0]).items() if isinstance(v, torch.Tensor)}
    (model.enable_hip_graphs if how == "graphs" else model.enable_launch_programs)(False)
    eager = run(frames[0])
    assert all(torch.equal(out[k], eager[k]) for k in KEYS) and not torch.equal(out[KEYS[0]], want[0][KEYS[0]])


def test_plane_statistics_of_a_hint_depth_with_per_pixel_planes():
    """The manager's method on a rendered depth map with holes, planes that vary over the image, and a mask."""
    model, frame, _, volume = _model(b=2)
    vol, _, planes, _ = volume(frame(4))
    g = torch.Generator().manual_seed(1)
    hint = torch.rand(2, 24, 32, generator=g) * 5
    hint[0, :4] = float("nan")
    hint[1, 5:9] = -1.0
    local = (planes * (0.9 + 0.2 * torch.rand(2, 1, 24, 32, generator=g)).to(vol.device)).contiguous()
    mask = (torch.rand(2, 1, 24, 32, generator=g) > 0.3).to(vol.device)
    r = model.cost_volume.plane_statistics(vol, local, hint.to(vol.device), top=2, mask_bdhw=mask)
    idx = ref.nearest(hint, local)
    assert bool((idx[0, :4] == -1).all()) and bool((idx[1, 5:9] == -1).all())
    ref.check_stats(r, vol, idx, 2, 1.0, mask, local)


def test_loop_masks_improbable_depths():
    from doubletake_amd import loops

    model, frame, run, _ = _model(b=2)
    out = run(frame(6))
    with pytest.raises(ValueError):
        loops._depth_for_fusion(out, None, min_plane_log_prob=-3.0)
    model.enable_plane_statistics(top=0)
    out = run(frame(6))
    lp = out["plane_log_prob_bhw"]
    thr = float(lp.median())
    depth = loops._depth_for_fusion(out, (96, 128), min_plane_log_prob=thr)
    keep = torch.nn.functional.interpolate((lp >= thr).float()[:, None], size=(96, 128), mode="nearest").bool()
    full = loops._depth_for_fusion(out, (96, 128))
    assert torch.equal(depth, torch.where(keep, full, torch.full_like(full, -1)))
    assert 0.3 < float(keep.float().mean()) < 0.7 and bool((full > 0).all())


def test_incremental_scan_fuses_less_with_a_threshold():
    import gpu_util as gu
    from doubletake_amd import loops
    from doubletake_amd.tools.fusers_helper import OurFuser

    bd = dict(xmin=-2.0, xmax=2.0, ymin=-2.0, ymax=2.0, zmin=0.0, zmax=2.4)
    h, w, k = 24, 32, 3
    H2, W2 = 2 * h, 2 * w
    model, _, _, _ = _model(b=1, h=h, w=w, k=k)
    model.enable_plane_statistics(top=0)
    tt = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(gu.dev())
    surface, K, T = syn.tsdf_frames(3, H2, W2, seed=11, bounds=bd)

    def scan(thr):
        batches = []
        for f in range(3):
            batches.append(({"K_s0_b44": tt(K[f:f + 1]), "invK_s0_b44": tt(np.linalg.inv(K[f:f + 1])), "cam_T_world_b44": tt(T[f:f + 1]),
                             "world_T_cam_b44": tt(np.linalg.inv(T[f:f + 1]).astype(np.float32)), "K_full_depth_b44": tt(K[f:f + 1]),
                             "f": f}, {}))

        def model_fn(cur, src):
            f = cur["f"]
            t = gu.to_dev(syn.volume_inputs(1, k, h, w, 16, f))
            pyr = [tt(p).contiguous(memory_format=torch.channels_last) for p in syn.prior_pyramid(1, [64, 64, 128, 256, 512], H2, W2, f)]
            out = dict(model.forward_from_features(pyr, t["cur_feats"], t["src_feats"], t["src_extrinsics"], t["src_poses"], t["src_Ks"],
                                                   t["cur_invK"], cur, return_mask=True))
            out["depth_pred_s0_b1hw"] = tt(surface[f:f + 1] * np.float32(0.6)).view(1, 1, H2, W2)
            return out

        fuser = OurFuser(None, 0.04, 3.0, bounds=bd)
        assert loops.run_incremental_scan(model_fn, fuser, batches, (H2, W2), min_plane_log_prob=thr) == 3
        return int((fuser.tsdf_fuser_pred.tsdf.tsdf_weights > 0).sum())

    everything, some, nothing = scan(None), scan(-2.7), scan(0.5)
    assert everything > 500 and nothing == 0 and nothing < some < everything
    assert scan(float("-inf")) == everything


def test_losses_on_the_volume_reach_the_features():
    """Training on the volume: a differentiable volume (torch products of matching features), a depth map's planes as targets,
    negative log likelihood and entropy; the features' gradients against the same loss in torch."""
    g = torch.Generator().manual_seed(3)
    b, C, D, h, w = 2, 8, 24, 6, 10
    cur = torch.randn(b, C, h, w, generator=g).cuda()
    warped = torch.randn(b, C, D, h, w, generator=g).cuda()
    planes = (0.25 * 20.0 ** torch.linspace(0, 1, D)).view(1, D, 1, 1).cuda()
    depth = (0.2 + 5 * torch.rand(b, h, w, generator=g)).cuda()
    depth[0, 0] = float("nan")

    def loss(c, own):
        vol = (c[:, :, None] * warped.to(c.dtype)).sum(1)
        idx = plane_ops.nearest_planes(depth, planes)
        ok = idx >= 0
        if own:
            r = plane_ops.plane_log_probs(vol, idx)
            return (-r.log_prob_bhw.sum() + 0.1 * r.entropy_bhw.sum()) / ok.sum()
        lp = torch.log_softmax(vol, 1)
        given = lp.gather(1, idx.clamp_min(0)[:, None])[:, 0] * ok
        return (-given.sum() - 0.1 * (lp.exp() * lp).sum()) / ok.sum()

    a = cur.clone().requires_grad_(True)
    loss(a, True).backward()
    e = cur.double().requires_grad_(True)
    loss(e, False).backward()
    # D products of gradient (error: a few float32 steps of values below 1.5 / 114 pixels ...) and feature (below 5), summed over D planes
    tol = D * 5 * (1.5 / 100) * 64 * 2.0 ** -24 + D * 5 * (1.5 / 100) * ref.bound_b(D)
    assert float((a.grad.double() - e.grad).abs().max()) < tol


def test_predictions_that_are_no_depth_are_not_certain():
    """NaN, infinite, zero and negative predictions fall on no plane: log probability -inf in the model's outputs, masked by the loops."""
    from doubletake_amd import loops

    model, frame, run, volume = _model(b=2)
    model.enable_plane_statistics(top=0)
    fr = frame(6)
    out = run(fr)
    vol, _, planes, _ = volume(fr)
    depth = out["depth_pred_s1_b1hw"].clone()
    bad = torch.zeros_like(depth, dtype=torch.bool)
    for k, v in enumerate((float("nan"), float("inf"), -float("inf"), 0.0, -1.0)):
        depth[:, :, k, 3:9] = v
        bad[:, :, k, 3:9] = True
    got = model._add_plane_statistics({"depth_pred_s1_b1hw": depth}, vol, planes)["plane_log_prob_bhw"]
    assert bool((got[bad[:, 0]] == -float("inf")).all())
    assert torch.equal(got[~bad[:, 0]], out["plane_log_prob_bhw"][~bad[:, 0]])
    full = loops._depth_for_fusion(dict(out, plane_log_prob_bhw=got), (24, 32), min_plane_log_prob=-1e30)
    assert bool((full[bad] == -1).all()) and bool((full[~bad] > 0).all())


def test_the_two_stages_driven_apart_equal_forward():
    model, frame, run, _ = _model(b=2)
    model.enable_plane_statistics(top=2)
    fr = frame(8)
    want = run(fr)
    seen = []
    kept = model.volume_stage
    model.volume_stage = lambda kw: seen.append(kw) or kept(kw)
    out = run(fr)
    assert len(seen) == 1 and all(torch.equal(out[k], want[k]) for k in KEYS)
    out = model.network_stage(fr[1], *kept(seen[0]))
    assert set(out) == set(want)
    for k, v in want.items():
        assert torch.equal(out[k], v), k
