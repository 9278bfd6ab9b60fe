"""The residual-block norms and their gradients in 64 bits, each with a bound on what f32 arithmetic may be off by, for the tests of the
kernels.  First-order error propagation, u = 2^-24, every bound made from the values' own rows and columns:

  a row's sum of D terms passes at most 8 additions in a thread, 6 in a wave and 16 over waves: 32 u of the mean of the absolute terms;
  z = (f - mean) / s:  dz <= u [(K + 4) |z| + K (mean|f| / s) (1 + |z|)], K = 32 (the mean's error, the root of the sum of squares, two
    roundings), without the mean: u (K + 4) |z|; an error of f itself passes on as (df + mean df + |z| mean(|z| df)) / s;
  sigmoid by v_exp_f32 and v_rcp_f32 (an ulp each): its exponent is off by 1.3 |g| u, so s by s (1.3 |g| + 6) u;
  a column's sum over n rows: at most 64 + n / 256 additions in a row.
Products and sums of two numbers carry a rounding each.  A stored 16-bit value is off by half a step of the exact one's neighbourhood."""
import torch

U = 2.0 ** -24
K = 32
PARAMS = ("res_scale", "post_scale", "post_bias", "pre_scale", "pre_bias")


def _mean(x):
    return x.mean(-1, keepdim=True)


class _Norm:
    """z = Norm(v), its error `dz` where v is off by `dv`, and the way back."""

    def __init__(self, v, dv, kind, eps):
        rms = kind == "rms_norm"
        c = v if rms else v - _mean(v)
        self.rms, self.s = rms, torch.sqrt(_mean(c * c) + eps)
        self.z = z = c / self.s
        a = z.abs()
        mean_term = torch.zeros_like(self.s) if rms else K * _mean(v.abs()) / self.s
        self.dz = U * ((K + 4) * a + mean_term * (1 + a)) + (dv + (0.0 if rms else 1.0) * _mean(dv) + a * _mean(a * dv)) / self.s
        self.rel = (K / 2 + 4) * U + U * mean_term + _mean(a * dv) / self.s         # of 1 / s

    def back(self, g, dg):
        """(gradient of the input, its error) from that of z and its error"""
        z, a = self.z, self.z.abs()
        p, q = _mean(g * z), torch.zeros_like(self.s) if self.rms else _mean(g)
        dp = _mean(a * dg + g.abs() * self.dz) + (K + 2) * U * _mean((g * z).abs())
        dq = torch.zeros_like(self.s) if self.rms else _mean(dg) + (K + 2) * U * _mean(g.abs())
        inner = g - z * p - q
        d = dg + a * dp + p.abs() * self.dz + dq + 2 * U * (g.abs() + (z * p).abs() + q.abs())
        return inner / self.s, d / self.s + inner.abs() / self.s * (self.rel + 2 * U)


def block(x, f, gate, gate_act, p, kind, post, pre, eps, dy, dh):
    """{name: (value, bound)} of y, h and the gradients of x, f, gate and the parameters that are not None; dy or dh may be None."""
    d64 = lambda t: None if t is None else t.double()      # noqa: E731
    x, f, gate, dy, dh = (d64(t) for t in (x, f, gate, dy, dh))
    one, zero = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device), torch.zeros(x.shape[-1], dtype=torch.float64, device=x.device)
    rs, ps, pb, qs, qb = (d64(p[n]) if p[n] is not None else (zero if n.endswith("bias") else one) for n in PARAMS)
    none = torch.zeros_like(x)
    nf = _Norm(f, none, kind, eps) if post else None
    z, dz = (nf.z, nf.dz) if post else (f, none)
    n = z * ps + pb
    dn_ = ps.abs() * dz + 2 * U * ((ps * z).abs() + pb.abs())
    if gate_act == "none":
        act, slope, dact, dslope = torch.ones_like(x), none, none, none
    else:
        s, g = torch.sigmoid(gate), gate.abs()
        if gate_act == "sigmoid":
            act, slope, dslope = s, s * (1 - s), s * U * (3 * g + 16)
        else:
            act, slope, dslope = gate * s, s * (1 + gate * (1 - s)), s * U * ((1.5 * g + 8) * (1 + 2 * g) + 4)
        dact = act.abs() * (1.3 * g + 8) * U
    y = x + rs * act * n
    ey = U * y.abs() + rs.abs() * (act.abs() * dn_ + n.abs() * dact + 3 * U * (act * n).abs())
    got = {"y": (y, ey)}
    ny = _Norm(y, ey, kind, eps) if pre else None
    if pre:
        got["h"] = (ny.z * qs + qb, qs.abs() * ny.dz + 2 * U * ((qs * ny.z).abs() + qb.abs()))
    if dy is None and dh is None:
        return got
    e, de = (none, none) if dy is None else (dy, none)
    if dh is not None:
        back, dback = ny.back(dh * qs, U * (dh * qs).abs())
        e, de = e + back, dback + U * (e.abs() + (e + back).abs())
    dn, ddn = e * rs * act, rs.abs() * (act.abs() * de + e.abs() * dact) + 3 * U * (e * rs * act).abs()
    got["dx"] = (e, de)
    if gate_act != "none":
        got["dgate"] = (e * rs * n * slope, rs.abs() * ((n * slope).abs() * de + (e * slope).abs() * dn_ + (e * n).abs() * dslope)
                        + 4 * U * (e * rs * n * slope).abs())
    df, ddf = dn * ps, ps.abs() * ddn + U * (dn * ps).abs()
    got["df"] = nf.back(df, ddf) if post else (df, ddf)

    def column(name, t, dt):
        if p[name] is not None:
            got["d" + name] = (t.sum(0), dt.sum(0) + (64 + x.shape[0] / 256) * U * t.abs().sum(0))

    column("res_scale", e * act * n, (act * n).abs() * de + e.abs() * (act.abs() * dn_ + n.abs() * dact) + 2 * U * (e * act * n).abs())
    column("post_scale", dn * z, z.abs() * ddn + dn.abs() * dz + U * (dn * z).abs())
    column("post_bias", dn, ddn)
    if dh is not None:
        column("pre_scale", dh * ny.z, dh.abs() * ny.dz + U * (dh * ny.z).abs())
        column("pre_bias", dh, none)
    else:
        column("pre_scale", none, none)
        column("pre_bias", none, none)
    return got


def outside(got, want, half):
    """The first name whose value leaves its bound (or None), with by how much; `half`: half a step of the rows' type.  f16 has steps of
    2^-24 below 2^-14: half of one more."""
    for name, (w, bound) in want.items():
        g = got[name].detach().double()
        assert g.shape == w.shape, (name, g.shape, w.shape)
        step = half if w.dim() == 2 else U
        least = 2.0 ** -25 if step == 2.0 ** -11 else 1e-30
        over = (g - w).abs() - (bound + step * (w.abs() + bound) + least)
        if not bool((over <= 0).all()):              # a NaN too
            return name, float(over.max()), int((~(over <= 0)).sum()), w.numel()
    return None


# rows, columns, the gate's activation, parameters, strided rows: one wave to a row, several, the widths over 4096 that are read twice,
# and more rows than workgroups (the column sums walk)
SHAPES = [(3, 2, "silu", True, False), (5, 64, "sigmoid", True, False), (130, 128, "silu", True, True), (7, 333, "none", True, False),
          (33, 1024, "silu", True, False), (6, 1025, "sigmoid", True, True), (9, 4096, "silu", True, False), (2, 4095, "silu", True, False),
          (3, 8192, "sigmoid", True, False), (4, 5001, "none", True, True), (900, 4100, "silu", True, False), (300, 5001, "silu", True, True),
          (70, 8191, "sigmoid", True, True), (8000, 160, "silu", True, False), (5000, 700, "sigmoid", True, False), (50000, 96, "silu", True, False)]


def inputs(device, n, d, dtype, seed, gate_act, params, strided):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)

    def normal(*shape, dt=dtype, s=1.0):
        return (torch.randn(*shape, generator=gen, device=device) * s).to(dt)

    def rows(s=1.0):
        return normal(n, 2 * d + 3, s=s)[:, d:2 * d] if strided else normal(n, d, s=s)

    x = {"x": rows(2.0), "f": rows(0.7), "gate": rows() if gate_act != "none" else None, "dy": rows(), "dh": rows()}
    for name in PARAMS:
        x[name] = normal(d, dt=torch.float32, s=0.3) + (0.0 if name.endswith("bias") else 0.8) if params else None
    return x
