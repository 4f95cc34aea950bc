"""sandwich_norm on the GPU against its definition in 64 bits.

Bounds.  u is the half-step of the 16-bit type, 2^-8 (bf16) or 2^-11 (fp16).
A row's sum of squares takes at most 48 fp32 roundings in a chain, so its
reciprocal root is within 2^-18 relative, and so is every product with it;
outputs add their own rounding.  Gradients chain two such norms: 2^-16 of the
sum of the magnitudes of what is added, and T 2^-24 more for a sum over T rows.
"""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0**-8, HF: 2.0**-11}
TINY = {BF: 2.0**-133, HF: 2.0**-25}
EPS = 1e-6


def _case(B, S, D, dt, seed, alpha=1.25, mod=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(
        x=(2 * r(B, S, D)).to(dt), res=(3 * r(B, S, D)).to(dt), gate=(0.5 * r(B, D)).to(dt) if mod else None,
        post=1 + 0.1 * r(D), pre=1 + 0.1 * r(D), shift=(0.1 * r(B, D)).to(dt) if mod else None,
        scale=(1 + 0.1 * r(B, D)).to(dt) if mod else None, alpha=alpha,
        gh=(0.1 * r(B, S, D)).to(dt), gz=(0.1 * r(B, S, D)).to(dt))


def _call(c, fn=None):
    return (fn or afb.sandwich_norm)(c["x"], c["res"], c["gate"], c["post"], c["pre"], c["shift"], c["scale"], c["alpha"], EPS)


def _rms(v):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _row(v, fallback):
    return fallback if v is None else v.double()[:, None]


def _z64(c):
    return c["alpha"] * c["res"].double(), _row(c["gate"], 1.0) * _rms(c["x"].double()) * c["post"].double()


def _h64(c, z):
    return _rms(z.double()) * c["pre"].double() * _row(c["scale"], 1.0), _row(c["shift"], 0.0) + torch.zeros_like(z.double())


def _within(got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst ratio {(err / tol).max():.3g}"


SHAPES = [(1, 1, 8), (1, 1, 2048), (2, 3, 72), (3, 5, 256), (1, 7, 264), (2, 9, 512), (1, 4, 1024), (2, 33, 1032), (3, 11, 2048),
          (1, 6, 2056), (2, 5, 4096), (1, 700, 640), (5, 1, 1152), (3, 701, 264), (1, 2051, 2056), (2, 1030, 2048),
          (1, 2049, 4096), (150, 15, 72)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,S,D", SHAPES)
def test_forward(B, S, D, dt, cuda_dev):
    c = _case(B, S, D, dt, B + S + D)
    h, z = _call(c)
    a, b = _z64(c)
    _within(z, a + b, U[dt] * (a + b).abs() + 2.0**-18 * (a.abs() + b.abs()) + TINY[dt])
    a, b = _h64(c, z)
    _within(h, a + b, U[dt] * (a + b).abs() + 2.0**-18 * (a.abs() + b.abs()) + TINY[dt])


@pytest.mark.parametrize("B,S,D", [(2, 3, 72), (1, 9, 512), (2, 33, 1032), (1, 4, 4096)])
def test_forward_without_modulation(B, S, D, cuda_dev):
    c = _case(B, S, D, BF, 1, alpha=1.0, mod=False)
    h, z = _call(c)
    a, b = _z64(c)
    _within(z, a + b, U[BF] * (a + b).abs() + 2.0**-18 * (a.abs() + b.abs()))
    a, _ = _h64(c, z)
    _within(h, a, (U[BF] + 2.0**-18) * a.abs())


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,S,D", [(1, 1, 16), (2, 3, 144), (3, 5, 256), (2, 9, 512), (2, 33, 1040), (3, 11, 2048), (2, 5, 4096), (3, 701, 272),
                                   (2, 1030, 2048), (1, 2049, 4096)])
def test_codes_of_the_output(B, S, D, dt, cuda_dev):
    c = _case(B, S, D, dt, 7 + D)
    q, s, z = _call(c, afb.sandwich_norm_int8)
    assert torch.equal(z, _call(c)[1])
    a, b = _h64(c, z)
    h = (a + b).view(-1, D)
    err = 2.0**-18 * (a.abs() + b.abs()).view(-1, D)
    top = h.abs().amax(1, keepdim=True)
    _within(s, top / 127.0, err.amax(1, keepdim=True) / 127.0 + 2.0**-23 * top)
    _within(q.view(-1, D).double() * s.double(), h, 0.5001 * s.double() + 2 * err.amax(1, keepdim=True))


def _bwd64(c, z, gz):
    """Gradients and, for each, the sum of the magnitudes of its terms."""
    x, z, gh = c["x"].double(), z.double(), c["gh"].double()
    gz = torch.zeros_like(z) if gz is None else gz.double()
    gate, scale, post, pre = _row(c["gate"], 1.0), _row(c["scale"], 1.0), c["post"].double(), c["pre"].double()
    r1 = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    r2 = 1 / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS)
    xh, zh = x * r1, z * r2
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    p = gh * scale * pre
    dz = gz + r2 * (p - zh * mean(p * zh))
    mz = gz.abs() + r2 * (p.abs() + zh.abs() * mean((p * zh).abs()))
    m, mm = dz * gate * post, mz * (gate * post).abs() if isinstance(gate, torch.Tensor) else mz * post.abs()
    dx = r1 * (m - xh * mean(m * xh))
    mx = r1 * (mm + xh.abs() * mean(mm * xh.abs()))
    P, mP = (gh * zh).sum(1), (gh * zh).abs().sum(1)
    Q, mQ = (dz * xh).sum(1), (mz * xh.abs()).sum(1)
    g2, s2 = (gate[:, 0], scale[:, 0]) if isinstance(gate, torch.Tensor) else (torch.ones_like(P), torch.ones_like(P))
    return dict(dx=(dx, mx), dres=(c["alpha"] * dz, c["alpha"] * mz), dgate=(Q * post, mQ * post.abs()),
                dpost=((g2 * Q).sum(0), (g2.abs() * mQ).sum(0)), dpre=((s2 * P).sum(0), (s2.abs() * mP).sum(0)),
                dshift=(gh.sum(1), gh.abs().sum(1)), dscale=(P * pre, mP * pre.abs()))


def _check_bwd(got, want, dt, T):
    for (name, (w, mag)), t in zip(want.items(), got):
        u = 0.0 if t.dtype == torch.float32 else U[dt]
        _within(t, w, u * w.abs() + (2.0**-16 + T * 2.0**-24) * mag + TINY[dt])


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,S,D", SHAPES + [(2, 1500, 256), (70, 3, 128)])
def test_backward(B, S, D, dt, cuda_dev):
    c = _case(B, S, D, dt, 3 * S + D)
    z = _call(c)[1]
    for gz in (c["gz"], None):
        got = afb.sandwich_norm_bwd(c["gh"], gz, z, c["x"], c["gate"], c["post"], c["pre"], c["scale"], c["alpha"], EPS)
        _check_bwd(got, _bwd64(c, z, gz), dt, B * S)
    again = afb.sandwich_norm_bwd(c["gh"], None, z, c["x"], c["gate"], c["post"], c["pre"], c["scale"], c["alpha"], EPS)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # one fixed order


def test_backward_without_modulation(cuda_dev):
    c = _case(2, 37, 264, BF, 5, mod=False)
    z = _call(c)[1]
    got = afb.sandwich_norm_bwd(c["gh"], c["gz"], z, c["x"], None, c["post"], c["pre"], None, c["alpha"], EPS)
    _check_bwd(got, _bwd64(c, z, c["gz"]), BF, 74)


@pytest.mark.parametrize("mod", [True, False])
def test_autograd(mod, cuda_dev):
    c = _case(2, 19, 520, BF, 9, mod=mod)
    names = ["x", "res", "gate", "post", "pre", "shift", "scale"]
    leaves = [c[n].detach().requires_grad_(True) for n in names if c[n] is not None]
    it = iter(leaves)
    args = [next(it) if c[n] is not None else None for n in names]
    h, z = afb.sandwich_norm(*args, c["alpha"], EPS)
    grads = torch.autograd.grad((h, z), leaves, (c["gh"], c["gz"]))
    want = _bwd64(c, z.detach(), c["gz"])
    order = ["dx", "dres"] + (["dgate"] if mod else []) + ["dpost", "dpre"] + (["dshift", "dscale"] if mod else [])
    _check_bwd(grads, {n: want[n] for n in order}, BF, 38)
    (gx,) = torch.autograd.grad(afb.sandwich_norm(*args, c["alpha"], EPS)[0].float().square().sum(), leaves[0])
    assert torch.isfinite(gx.float()).all()


def test_backward_against_differences(cuda_dev):
    """Directional derivatives of the formula in 64 bits, z not rounded.

    The kernel's z differs from the unrounded one by u relative, which moves a
    gradient by a few u of its terms; the outputs add u: 8 u of the magnitudes.
    """
    c = _case(2, 5, 136, BF, 21)
    z = _call(c)[1]
    got = dict(zip(["x", "res", "gate", "post", "pre", "shift", "scale"],
                   afb.sandwich_norm_bwd(c["gh"], c["gz"], z, c["x"], c["gate"], c["post"], c["pre"], c["scale"], c["alpha"], EPS)))
    mags = dict(zip(["x", "res", "gate", "post", "pre", "shift", "scale"], _bwd64(c, z, c["gz"]).values()))

    def loss(d):
        e = {k: (v.double() if isinstance(v, torch.Tensor) else v) for k, v in c.items()} | d
        zz = sum(_z64(e))
        hh = _rms(zz) * e["pre"] * e["scale"][:, None] + e["shift"][:, None]
        return (hh * e["gh"] + zz * e["gz"]).sum()

    g = torch.Generator(device="cuda").manual_seed(1)
    for name, t in got.items():
        v = torch.randn(t.shape, generator=g, device=cuda_dev, dtype=torch.float64)
        d = 2.0**-16
        diff = (loss({name: c[name].double() + d * v}) - loss({name: c[name].double() - d * v})) / (2 * d)
        tol = 8 * U[BF] * (mags[name][1] * v.abs()).square().sum().sqrt() + 2.0**-20 * (mags[name][1] * v.abs()).sum()
        assert abs((t.double() * v).sum() - diff) <= tol, name


def test_zero_rows_and_non_finite_rows(cuda_dev):
    c = _case(1, 4, 256, BF, 2)
    c["x"][0, 0] = 0  # an empty token: its norm is zero, not NaN
    c["res"][0, 0] = 0
    c["x"][0, 2, 7] = float("inf")
    c["res"][0, 3, 9] = float("nan")
    h, z = _call(c)
    assert not z[0, 0].any() and torch.equal(h[0, 0], c["shift"][0])
    assert torch.isnan(h[0, 3].float()).all() and torch.isfinite(h[0, 1].float()).all()
    assert torch.isnan(z[0, 2, 7].float())
    q, s, _ = _call(c, afb.sandwich_norm_int8)
    assert torch.isfinite(s[1]) and not torch.isfinite(s[3]) and not q[0, 3].any()


def test_empty_and_strided(cuda_dev):
    c = _case(2, 0, 64, BF, 2)
    h, z = _call(c)
    assert h.shape == z.shape == (2, 0, 64)
    g = afb.sandwich_norm_bwd(c["gh"], None, z, c["x"], c["gate"], c["post"], c["pre"], c["scale"])
    assert g[0].shape == (2, 0, 64) and not any(t.any() for t in g[2:])
    c = _case(2, 9, 64, BF, 2)
    wide = torch.cat([c["x"], c["res"]], -1)
    h, z = _call(c)
    c["x"], c["res"] = wide[..., :64], wide[..., 64:]
    h2, z2 = _call(c)
    assert torch.equal(h, h2) and torch.equal(z, z2)
