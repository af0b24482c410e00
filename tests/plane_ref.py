"""Plain 64-bit forms of doubletake_amd.modules.plane_ops and the error bounds of its 32-bit arithmetic (tests only).

u = 2^-24 is half a float32 step.  With y = scale (x - max) every term e = exp(y) of the sum s carries a relative error of at most
4 u |y| (rounding of the difference, of the product and of the folded constant) + 4 u (the exponential); sum e |y| / s = H - ln s <= ln D
and s itself D roundings, so that
    |ln s - exact|    <= u (D + 16 + 6 ln D)                                  =: A
    |log_prob - exact| <= A + 4 u |log_prob|                                   (|y| <= |log_prob|)
    |entropy - exact|  <= A + u ((D + 16) ln D + 4 ((ln D)^2 + 2))             =: B
      (H = ln s + sum e |y| / s; sum e y^2 / s <= (ln D)^2 + 2)
"""
import math

import numpy as np
import torch

U = 2.0 ** -24


def bound_a(D):
    return U * (D + 16 + 6 * math.log(D))


def bound_b(D):
    return bound_a(D) + U * ((D + 16) * math.log(D) + 4 * (math.log(D) ** 2 + 2))


def stats(vol, plane=None, top=0, scale=1.0, mask=None, planes=None):
    """dict of float64 / int64 CPU tensors; vol may be any float type and device, differentiable if it is a float64 leaf."""
    x = vol.cpu().double()
    b, D, h, w = x.shape
    z = x * float(np.float32(scale))
    if mask is not None:
        z = z.masked_fill(~mask.cpu().expand(x.shape), -math.inf)
    m = z.detach().amax(1, keepdim=True)
    m0 = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(z - m0)
    e = torch.where(z == -math.inf, torch.zeros_like(e), e)
    s = e.sum(1, keepdim=True)
    empty = s == 0
    ls = torch.log(torch.where(empty, torch.ones_like(s), s))
    seen = z != -math.inf
    lp = torch.where(seen, z - m0, torch.zeros_like(z)) - ls
    p = e / torch.where(empty, torch.ones_like(s), s)
    ninf = torch.full_like(lp, -math.inf)
    lp_all = torch.where(seen, lp, ninf)
    out = {"entropy": -(p * torch.where(seen, lp, torch.zeros_like(lp))).sum(1),
           "log_sum": torch.where(empty, torch.full_like(s, -math.inf), m0 + ls)[:, 0]}
    if plane is not None:
        idx = plane.cpu().long()
        ok = (idx >= 0) & (idx < D)
        v = lp_all.gather(1, torch.where(ok, idx, torch.zeros_like(idx))[:, None])[:, 0]
        out["log_prob"] = torch.where(ok, v, torch.zeros_like(v))
    if top:
        zn = z.detach().numpy()
        # NaN first, then by score, then by plane: lexsort's last key is the primary one
        order = np.lexsort((np.broadcast_to(np.arange(D)[None, :, None, None], zn.shape), np.where(np.isnan(zn), 0.0, -zn),
                            ~np.isnan(zn)), axis=1)[:, :top]
        order = torch.from_numpy(np.ascontiguousarray(order))
        v = lp_all.gather(1, order)
        have = z.detach().gather(1, order) != -math.inf
        out["top_log_prob"] = torch.where(have, v, torch.full_like(v, -math.inf))
        out["top_plane"] = torch.where(have, order, torch.full_like(order, -1))
        if planes is not None:
            dep = planes.cpu().expand(x.shape).gather(1, order)
            out["top_depth"] = torch.where(have, dep, torch.zeros_like(dep))
    out["p"], out["lp"] = p.detach(), torch.where(seen, lp, torch.zeros_like(lp)).detach()
    return out


def close(got, want, atol, rtol=0.0, what=""):
    got = got.detach().cpu().double()
    want = want.detach().double()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.float().double(), want)   # (-6.8e38 is -inf in float32)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    same = torch.where(torch.isnan(want), torch.isnan(got), got == want)
    assert bool(same[~fine].all()), f"{what}: infinities / NaN differ"
    assert bool(torch.isfinite(got)[fine].all()), f"{what}: not finite where it should be"
    over = (got - want).abs()[fine] - (atol[fine] if isinstance(atol, torch.Tensor) else atol) - rtol * want.abs()[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: over the bound by {float(over.max()):.3e}"


def check_stats(res, vol, plane=None, top=0, scale=1.0, mask=None, planes=None):
    D = vol.shape[1]
    ref = stats(vol.detach(), plane, top, scale, mask, planes)
    a, b = bound_a(D), bound_b(D)
    close(res.entropy_bhw, ref["entropy"], b, 0.0, "entropy")
    big = torch.where(torch.isfinite(ref["log_sum"]), ref["log_sum"].abs() + math.log(D), torch.zeros_like(ref["log_sum"]))
    close(res.log_sum_bhw, ref["log_sum"], a + 4 * U * big, 0.0, "log_sum")
    if plane is not None:
        close(res.log_prob_bhw, ref["log_prob"], a, 4 * U, "log_prob")
    else:
        assert res.log_prob_bhw is None
    if top:
        assert torch.equal(res.top_plane_bkhw.cpu(), ref["top_plane"]), "top_plane"
        close(res.top_log_prob_bkhw, ref["top_log_prob"], a, 4 * U, "top_log_prob")
        if planes is not None:
            assert torch.equal(res.top_depth_bkhw.cpu(), ref["top_depth"]), "top_depth"
    else:
        assert res.top_log_prob_bkhw is None and res.top_plane_bkhw is None
    return ref


def gradient(vol, plane, top, scale, mask, g_lp=None, g_ent=None, g_lsum=None, g_top=None):
    """float64 gradient of the volume by the formula, and the bound of its error before the last rounding."""
    ref = stats(vol.detach(), plane, top, scale, mask)
    D = vol.shape[1]
    p, lp, ent = ref["p"], ref["lp"], ref["entropy"][:, None]
    cpu = lambda g: None if g is None else g.detach().cpu().double()
    g_lp, g_ent, g_lsum, g_top = cpu(g_lp), cpu(g_ent), cpu(g_lsum), cpu(g_top)
    total, size = torch.zeros_like(ent), torch.zeros_like(ent)
    hits, hits_size = torch.zeros_like(p), torch.zeros_like(p)
    if g_lsum is not None:
        total, size = total + g_lsum[:, None], size + g_lsum[:, None].abs()
    if g_lp is not None:
        idx = plane.cpu().long()
        ok = (idx >= 0) & (idx < D)
        g = torch.where(ok, g_lp, torch.zeros_like(g_lp))[:, None]
        total, size = total - g, size + g.abs()
        hits.scatter_add_(1, torch.where(ok, idx, torch.zeros_like(idx))[:, None], g)
        hits_size.scatter_add_(1, torch.where(ok, idx, torch.zeros_like(idx))[:, None], g.abs())
    if g_top is not None:
        have = ref["top_plane"] >= 0
        g = torch.where(have, g_top, torch.zeros_like(g_top))
        total, size = total - g.sum(1, keepdim=True), size + g.abs().sum(1, keepdim=True)
        hits.scatter_add_(1, ref["top_plane"].clamp_min(0), g)
        hits_size.scatter_add_(1, ref["top_plane"].clamp_min(0), g.abs())
    # (d lp_g / dx_g = 1 - p_g holds for every finite score, also where p_g underflows; a score of -inf has no derivative)
    seen = vol.detach().cpu() != -math.inf
    if mask is not None:
        seen = seen & mask.cpu().expand(seen.shape)
    hits, hits_size = torch.where(seen, hits, torch.zeros_like(hits)), torch.where(seen, hits_size, torch.zeros_like(hits))
    ge = torch.zeros_like(ent) if g_ent is None else g_ent[:, None]
    sc = float(np.float32(scale))
    grad = sc * (hits + p * (total - ge * (lp + ent)))
    # p: relative error of exp(lp), lp off by A + 4 u |lp|; the bracket's own terms; about ten roundings of sums and products.  The
    # sum of a given plane's and the alternatives' gradients that meet one plane rounds at every partial sum, each of which is as
    # large as the sum of the ABSOLUTE values, not as the result: +1 - 1 + 1e-3 is off by u, not by 1e-3 u
    eps = bound_a(D) + U * (4 * lp.abs() + 8)
    err = sc * (p * (eps + 16 * U) * (size + ge.abs() * (lp.abs() + ent)) + p * ge.abs() * (eps + bound_b(D))
                + 16 * U * (hits_size + p * size))
    return grad, err


def nearest(depth, planes):
    """int64 [b,h,w] by a loop over planes in 64 bits."""
    dep = depth.cpu().float().double()
    pl = planes.cpu().double()
    best = torch.full_like(dep, math.inf)
    at = torch.full(dep.shape, -1, dtype=torch.int64)
    for d in range(pl.shape[1]):
        off = (pl[:, d].expand(dep.shape) - dep).abs()
        take = off < best
        best = torch.where(take, off, best)
        at[take] = d
    at[~(torch.isfinite(dep) & (dep > 0))] = -1
    return at
