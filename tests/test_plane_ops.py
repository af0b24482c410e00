"""plane_ops on the CPU: every refusal comes before a launch, and the 64-bit form the GPU tests compare with is itself checked
against torch's log_softmax and against differences."""
import ctypes as C
import math
import types

import pytest
import torch

import plane_ref as ref
from doubletake_amd import _abi
from doubletake_amd.modules import plane_ops


def _vol(b=2, D=5, h=3, w=4, dtype=torch.float32):
    return torch.zeros(b, D, h, w, dtype=dtype)


def _refusals():
    v = _vol()
    i = torch.zeros(2, 3, 4, dtype=torch.int64)
    m = torch.ones(2, 5, 3, 4, dtype=torch.bool)
    p = torch.ones(2, 5, 3, 4)
    return {
        "3-D volume": (v[0], {}),
        "double volume": (v.double(), {}),
        "integer volume": (v.long(), {}),
        "no planes": (v[:, :0], {}),
        "top over D": (v, dict(top=6)),
        "top over 8": (_vol(D=20), dict(top=9)),
        "top negative": (v, dict(top=-1)),
        "scale zero": (v, dict(scale=0.0)),
        "scale negative": (v, dict(scale=-1.0)),
        "scale nan": (v, dict(scale=math.nan)),
        "scale inf": (v, dict(scale=math.inf)),
        "scale too large": (v, dict(scale=2e30)),
        "scale too small": (v, dict(scale=1e-31)),
        "too many planes": (torch.zeros(1).expand(1, (1 << 30) + 1, 1, 1), {}),
        "plane float": (v, dict(plane_bhw=i.float())),
        "plane shape": (v, dict(plane_bhw=i[:, None])),
        "plane size": (v, dict(plane_bhw=i[:1])),
        "mask type": (v, dict(mask_bdhw=m.float())),
        "mask dims": (v, dict(mask_bdhw=m[0])),
        "mask size": (v, dict(mask_bdhw=m[:, :4])),
        "planes without top": (v, dict(depth_planes_bdhw=p)),
        "planes type": (v, dict(depth_planes_bdhw=p.double(), top=1)),
        "planes size": (v, dict(depth_planes_bdhw=p[:, :, :2], top=1)),
    }


@pytest.mark.parametrize("name", sorted(_refusals()))
def test_plane_log_probs_refuses(name):
    vol, kw = _refusals()[name]
    with pytest.raises(ValueError):
        plane_ops.plane_log_probs(vol, **kw)


def test_too_many_pixels_are_refused():
    big = torch.zeros(1).expand(2, 3, 1 << 15, 1 << 15)
    with pytest.raises(ValueError, match="pixels"):
        plane_ops.plane_log_probs(big)
    with pytest.raises(ValueError, match="pixels"):
        plane_ops.nearest_planes(big[:, 0], torch.ones(1, 3, 1, 1))


def test_no_cpu_fallback():
    with pytest.raises(_abi.DoubletakeHipError):
        plane_ops.plane_log_probs(_vol())
    with pytest.raises(_abi.DoubletakeHipError):
        plane_ops.nearest_planes(torch.ones(2, 3, 4), torch.ones(2, 5, 1, 1))


@pytest.mark.parametrize("depth,planes", [
    (torch.ones(2, 1, 3, 4), torch.ones(2, 5, 1, 1)),
    (torch.ones(2, 3, 4, dtype=torch.int64), torch.ones(2, 5, 1, 1)),
    (torch.ones(2, 3, 4), torch.ones(2, 5)),
    (torch.ones(2, 3, 4), torch.ones(2, 0, 1, 1)),
    (torch.ones(2, 3, 4), torch.ones(2, 5, 1, 1, dtype=torch.float64)),
    (torch.ones(2, 3, 4), torch.ones(3, 5, 1, 1)),
    (torch.ones(2, 3, 4), torch.ones(2, 5, 3, 3)),
])
def test_nearest_planes_refuses(depth, planes):
    with pytest.raises(ValueError):
        plane_ops.nearest_planes(depth, planes)


def _desc(**kw):
    d = _abi.PlaneDesc()
    vals = dict(b=1, d=4, h=2, w=2, dtype=0, top=0, scale=1.0)
    vals.update(kw)
    for k, v in vals.items():
        setattr(d, k, v)
    return d


def _call(d, **kw):
    a = dict(volume=16, mask=None, plane=None, planes=None, log_prob=None, entropy=16, log_sum=16, tlp=None, tpl=None, tdep=None,
             rmax=None, rlog=None)
    a.update(kw)
    return _abi.lib().dt_cv_plane_log_probs(C.byref(d) if d is not None else None, *a.values(), None)


def _call_grad(d, **kw):
    a = dict(volume=16, mask=None, plane=None, entropy=16, tpl=None, rmax=16, rlog=16, g_lp=None, g_ent=None, g_lsum=None, g_top=None,
             grad=16)
    a.update(kw)
    return _abi.lib().dt_cv_plane_log_probs_grad(C.byref(d) if d is not None else None, *a.values(), None)


@pytest.mark.parametrize("bad", [dict(b=0), dict(d=0), dict(h=-1), dict(w=0), dict(dtype=3), dict(dtype=-1), dict(top=5), dict(top=9, d=20),
                                 dict(top=-1), dict(scale=0.0), dict(scale=-2.0), dict(scale=math.inf), dict(scale=math.nan),
                                 dict(scale=2e30), dict(scale=1e-31), dict(d=(1 << 30) + 1),
                                 dict(vol_stride=(C.c_int64 * 4)(1, -1, 1, 1)), dict(mask_stride=(C.c_int64 * 4)(1, 1, -1, 1)),
                                 dict(planes_stride=(C.c_int64 * 4)(-1, 1, 1, 1)), dict(grad_stride=(C.c_int64 * 4)(1, 1, 1, -1)),
                                 dict(b=1 << 15, h=1 << 15, w=2)])
def test_abi_refuses_descriptors(bad):
    assert _call(_desc(**bad)) != 0 and _abi.lib().dt_last_error()
    assert _call_grad(_desc(**bad)) != 0


def test_abi_refuses_pointers():
    assert _call(None) != 0 and _call_grad(None) != 0
    for kw in (dict(volume=None), dict(entropy=None), dict(log_sum=None), dict(plane=16), dict(log_prob=16), dict(rmax=16),
               dict(rlog=16), dict(tdep=16), dict(tdep=16, planes=16)):
        assert _call(_desc(), **kw) != 0, kw
    assert _call(_desc(top=2)) != 0 and _call(_desc(top=2), tlp=16) != 0
    for kw in (dict(volume=None), dict(entropy=None), dict(rmax=None), dict(rlog=None), dict(grad=None), dict(g_lp=16),
               dict(g_top=16), dict(g_top=16, tpl=16)):
        assert _call_grad(_desc(), **kw) != 0, kw
    L, st = _abi.lib(), (C.c_int64 * 4)(4, 1, 0, 0)
    for args in ((None, 16, st, 1, 4, 2, 2, 16), (16, None, st, 1, 4, 2, 2, 16), (16, 16, None, 1, 4, 2, 2, 16), (16, 16, st, 1, 4, 2, 2, None),
                 (16, 16, (C.c_int64 * 4)(4, 1, -1, 0), 1, 4, 2, 2, 16), (16, 16, st, 1, (1 << 30) + 1, 2, 2, 16), (16, 16, st, 0, 4, 2, 2, 16), (16, 16, st, 1, 0, 2, 2, 16), (16, 16, st, 1 << 15, 4, 1 << 15, 2, 16)):
        assert L.dt_cv_nearest_planes_f32(*args, None) != 0, args


def test_reference_form_matches_log_softmax():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 9, 4, 5, generator=g, dtype=torch.float64)
    idx = torch.randint(0, 9, (2, 4, 5), generator=g)
    r = ref.stats(x, idx, top=3, scale=0.5)
    lp = torch.log_softmax(x * 0.5, 1)
    assert torch.allclose(r["log_prob"], lp.gather(1, idx[:, None])[:, 0], atol=1e-14)
    assert torch.allclose(r["entropy"], -(lp.exp() * lp).sum(1), atol=1e-14)
    assert torch.allclose(r["log_sum"], torch.logsumexp(x * 0.5, 1), atol=1e-14)
    v, i = torch.topk(lp, 3, dim=1)
    assert torch.equal(r["top_plane"], i) and torch.allclose(r["top_log_prob"], v, atol=1e-14)


def test_reference_gradient_matches_autograd_and_differences():
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, idx = rnd(1, 6, 2, 3), torch.randint(-1, 6, (1, 2, 3), generator=g)
    mask = torch.rand(1, 6, 2, 3, generator=g) > 0.3
    mask[0, :, 0, 0] = False
    gl, ge, gs, gt = rnd(1, 2, 3), rnd(1, 2, 3), rnd(1, 2, 3), rnd(1, 2, 2, 3)
    idx = torch.where(mask.gather(1, idx.clamp_min(0)[:, None])[:, 0], idx, torch.full_like(idx, -1))

    def loss(v):
        r = ref.stats(v, idx, 2, 2.0, mask)
        fin = lambda t: torch.where(torch.isfinite(t), t, torch.zeros_like(t))
        return (fin(r["log_prob"]) * gl + r["entropy"] * ge + fin(r["log_sum"]) * gs).sum() + (fin(r["top_log_prob"]) * gt).sum()

    leaf = x.clone().requires_grad_(True)
    auto, = torch.autograd.grad(loss(leaf), leaf)
    want, _ = ref.gradient(x, idx, 2, 2.0, mask, gl, ge, gs, gt)
    assert torch.allclose(want, torch.nan_to_num(auto), atol=1e-12)
    eps = 1e-5
    for k in range(x.numel()):
        d = torch.zeros_like(x)
        d.view(-1)[k] = eps
        assert abs(float((loss(x + d) - loss(x - d)) / (2 * eps) - want.view(-1)[k])) < 1e-7


def test_model_refuses_bad_statistics_settings_and_loops_need_them():
    from doubletake_amd import loops
    from doubletake_amd.experiment_modules.doubletake_model import DepthModelCVHint

    m = DepthModelCVHint(64, 96, matching_num_depth_bins=6, model_num_views=3, matching_encoder_type=None)
    for kw in (dict(top=7), dict(top=-1), dict(scale=0.0), dict(scale=math.inf), dict(scale=math.nan)):
        with pytest.raises(ValueError):
            m.enable_plane_statistics(**kw)
    assert m.enable_plane_statistics(top=6) is m and m._launch_config() != m.enable_plane_statistics(False)._launch_config()
    depth = torch.ones(1, 1, 4, 6)
    with pytest.raises(ValueError, match="enable_plane_statistics"):
        loops._depth_for_fusion({"depth_pred_s0_b1hw": depth}, None, min_plane_log_prob=-1.0)
    lp = torch.tensor([[[-0.5, -2.0, math.nan], [-1.0, 0.0, -math.inf]]])
    got = loops._depth_for_fusion({"depth_pred_s0_b1hw": depth, "plane_log_prob_bhw": lp}, None, min_plane_log_prob=-1.0)
    want = torch.tensor([[1.0, -1, -1], [1, 1, -1]]).repeat_interleave(2, 0).repeat_interleave(2, 1)
    assert torch.equal(got[0, 0], want) and bool((depth == 1).all())


def _saved(**kw):
    """What a backward pass of a [2, 5, 3, 4] volume with a mask, given planes and two alternatives finds saved."""
    b, D, h, w, top = 2, 5, 3, 4, 2
    t = dict(vol=torch.zeros(b, D, h, w), plane=torch.zeros(b, h, w, dtype=torch.int64), mask=torch.ones(b, D, h, w, dtype=torch.bool),
             ent=torch.zeros(b, h, w), tpl=torch.zeros(b, top, h, w, dtype=torch.int64))
    ctx = types.SimpleNamespace(rows=torch.zeros(2, b, h, w), stream=None, top=top, scale=1.0, dtype=torch.float32,
                                shape=t["vol"].shape, vol_stride=t["vol"].stride(), mask_stride=t["mask"].stride(),
                                desc=plane_ops._desc(t["vol"], top, 1.0, t["mask"], None))
    t.update(kw)
    ctx.saved_tensors = tuple(t.values())
    return ctx


@pytest.mark.parametrize("name,bring", [
    ("vol", lambda t: t.half()), ("vol", lambda t: t[:, :4]), ("vol", lambda t: t.to("meta")),
    ("plane", lambda t: t.int()), ("plane", lambda t: t.to("meta")), ("plane", lambda t: t[:1]),
    ("mask", lambda t: t.float()), ("mask", lambda t: t[:, :1]), ("mask", lambda t: t.to("meta")),
    ("ent", lambda t: t.half()), ("ent", lambda t: t[0]), ("tpl", lambda t: t.int()), ("tpl", lambda t: t[:, :1])])
def test_backward_refuses_saved_tensors_brought_back_as_others(name, bring, monkeypatch):
    """A hook on saved tensors returned another device, type or size: refused before the kernel is given an address."""
    calls = []

    class Lib:
        def dt_cv_plane_log_probs_grad(self, *a):
            calls.append(a)
            return 0

    monkeypatch.setattr(_abi, "lib", Lib)
    g = torch.ones(2, 3, 4)
    good = _saved()
    assert plane_ops._backward(good, g, g, g, torch.ones(2, 2, 3, 4), None, None)[0].shape == good.shape and len(calls) == 1
    order = ("vol", "plane", "mask", "ent", "tpl")
    bad = _saved(**{name: bring(good.saved_tensors[order.index(name)])})
    with pytest.raises(RuntimeError, match="hook on saved tensors"):
        plane_ops._backward(bad, g, g, g, torch.ones(2, 2, 3, 4), None, None)
    assert len(calls) == 1


def test_planes_that_float32_sums_do_not_bear_are_refused():
    """More than 65536 planes: with float32 sums the normaliser would be off by 1e-3 and more, and stop growing at 2^24 of them."""
    shape = lambda D: torch.zeros(1).expand(1, D, 1, 1)
    for D in ((1 << 16) + 1, 1 << 20, 1 << 24):
        with pytest.raises(ValueError, match="planes"):
            plane_ops.plane_log_probs(shape(D))
        assert _call(_desc(d=D)) != 0 and _call_grad(_desc(d=D)) != 0
    with pytest.raises(_abi.DoubletakeHipError, match="CPU"):   # (accepted as far as the device)
        plane_ops.plane_log_probs(shape(1 << 16))
    with pytest.raises(_abi.DoubletakeHipError, match="CPU"):   # (a search sums nothing)
        plane_ops.nearest_planes(torch.ones(1, 1, 1), shape(1 << 24))


@pytest.mark.parametrize("size", [None, (4, 6)])
def test_loops_mask_predictions_that_are_no_depth(size):
    """A log probability of 0 (what an operator reports for a pixel without a plane) does not make a NaN or infinite depth certain."""
    from doubletake_amd import loops

    depth = torch.tensor([[1.0, math.nan, math.inf], [-math.inf, 0.0, -2.0]]).view(1, 1, 2, 3)
    got = loops._depth_for_fusion({"depth_pred_s0_b1hw": depth, "plane_log_prob_bhw": torch.zeros(1, 2, 3)}, size, min_plane_log_prob=-1.0)
    want = torch.tensor([[1.0, -1, -1], [-1, -1, -1]]).view(1, 1, 2, 3)
    if size:
        want = want.repeat_interleave(2, 2).repeat_interleave(2, 3)
    assert torch.equal(got, want)


@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_tangents_are_refused(needs_grad):
    """They would be dropped without a word; the volume without one is taken as ever (as far as the device, here)."""
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        v = _vol()
        dual = forward_ad.make_dual(v.requires_grad_(needs_grad), torch.ones_like(v))
        with pytest.raises(NotImplementedError, match="tangent"):
            plane_ops.plane_log_probs(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
            plane_ops.plane_log_probs(dual)
        with pytest.raises(_abi.DoubletakeHipError):
            plane_ops.plane_log_probs(_vol())
    with pytest.raises(NotImplementedError, match="tangent"):
        torch.func.jvp(lambda x: plane_ops.plane_log_probs(x).entropy_bhw, (_vol(),), (_vol(),))


def _staged_model(calls, monkeypatch):
    """A model on the CPU whose volume, network and statistics only report their calls."""
    from doubletake_amd.experiment_modules.doubletake_model import DepthModelCVHint

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)   # (torch asks a device otherwise)
    m = DepthModelCVHint(64, 96, matching_num_depth_bins=6, model_num_views=3, matching_encoder_type=None)
    vol, planes, depth = torch.zeros(1, 6, 16, 24), torch.ones(1, 6, 16, 24), torch.ones(1, 1, 16, 24)

    def statistics(cost_volume, depth_planes_bdhw, depth_bhw, top=0, scale=1.0, **kw):
        calls.append(("statistics", cost_volume, depth_planes_bdhw))
        z = torch.zeros(1, 16, 24)
        return plane_ops.PlaneLogProbs(z, z, z, None, None, None)

    m.cost_volume.forward = lambda **kw: calls.append(("volume",)) or (vol, vol[:, 0], planes, None)
    m.cost_volume.plane_statistics = statistics
    m.cost_volume_net.forward = lambda *a: []
    m.depth_decoder.forward = lambda *a, **kw: {"log_depth_pred_s1_b1hw": torch.zeros_like(depth), "depth_pred_s1_b1hw": depth}
    run = lambda: m.forward_from_features([None] * 5, torch.zeros(1, 16, 16, 24), torch.zeros(1, 2, 16, 16, 24), None, None, None, None, {})
    return m, run, vol, planes


def test_the_volume_stage_is_the_way_to_the_volume_with_statistics_too(monkeypatch):
    calls = []
    m, run, vol, planes = _staged_model(calls, monkeypatch)
    own_vol, own_planes = vol + 1, planes + 1
    for on in (False, True):
        m.enable_plane_statistics(on, top=0)
        calls.clear()
        assert ("plane_log_prob_bhw" in run()) is on
        assert [c[0] for c in calls] == ["volume", "statistics"][:1 + on]
        if on:
            assert calls[1][1] is vol and calls[1][2] is planes
        # a replaced stage is used, with its own planes
        m.volume_stage = lambda kw: calls.append(("stage",)) or ((own_vol, None, None, own_planes) if on else (own_vol, None, None))
        calls.clear()
        assert ("plane_log_prob_bhw" in run()) is on
        assert [c[0] for c in calls] == ["stage", "statistics"][:1 + on]
        if on:
            assert calls[1][1] is own_vol and calls[1][2] is own_planes
            m.volume_stage = lambda kw: (own_vol, None, None)
            with pytest.raises(ValueError, match="volume_stage returns"):
                run()
        del m.volume_stage
        # a replaced network stage takes what it always took
        m.network_stage = lambda cur_feats, cost_volume, lowest_cost, overall_mask: {"depth_pred_s1_b1hw": torch.ones(1, 1, 16, 24)}
        assert ("plane_log_prob_bhw" in run()) is on
        del m.network_stage


def test_the_two_stages_driven_apart_yield_statistics(monkeypatch):
    calls = []
    m, run, vol, planes = _staged_model(calls, monkeypatch)
    assert len(m.volume_stage({})) == 3 and "plane_log_prob_bhw" not in m.network_stage([None] * 5, *m.volume_stage({}))
    m.enable_plane_statistics(top=0)
    stage = m.volume_stage({})
    assert len(stage) == 4
    out = m.network_stage([None] * 5, *stage)
    assert "plane_log_prob_bhw" in out and set(out) == set(run())
    assert "plane_log_prob_bhw" not in m.network_stage([None] * 5, *stage[:3])
    m.enable_plane_statistics(False)
    assert "plane_log_prob_bhw" not in m.network_stage([None] * 5, *stage)


def test_header_states_which_outputs_go_together():
    """The refusals of test_abi_refuses_pointers, as a C caller reads them."""
    import os
    import re

    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "doubletake_hip.h")).read()
    words = re.sub(r"[\s*]+", " ", text[text.index("Statistics of every pixel"):text.index("int dt_cv_plane_log_probs(")])
    assert "may be NULL where it is not wanted" not in words
    for says in ("log_prob [b,h,w] goes with plane_bhw: both or neither", "top_log_prob and top_plane [b,top,h,w] are both required",
                 "top_depth [b,top,h,w] may be NULL and needs depth_planes", "row_max and row_log [b,h,w], both or neither"):
        assert says in words, says


def test_gradients_that_torch_negates_when_read():
    g = torch.tensor([[[2.0]]])
    lazy = torch.complex(torch.zeros_like(g), -g).conj().imag
    assert lazy.is_neg() and lazy.is_contiguous()
    got = plane_ops._dense_f32(lazy)
    assert not got.is_neg() and torch.equal(got, g) and plane_ops._dense_f32(g) is g and plane_ops._dense_f32(None) is None
