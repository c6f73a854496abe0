"""Per-head q / k norms with the position rotation and attention with a bucketed relative position bias, against their
definitions in 64 bits.  CPU: host emulation of the kernel sources; -m gpu: gfx950 library.

Tolerances are worst-case bounds formed from the inputs (u = 2^-24 a 32-bit rounding, 2^-8 a bf16 rounding): every sum of n
terms is off by at most (n + a few) u times the sum of magnitudes, every rounding to bf16 by 2^-8 of the value."""
import math

import pytest
import torch

from occformer_amd.ops import OccfError
from occformer_amd.position import RelativeBuckets, rotary_table

U = 2.0 ** -24
BF = 2.0 ** -8
NAN = float("nan")


def _randn(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def _half(dtype):
    return BF if dtype == torch.bfloat16 else U


def _within(got, ref, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst ratio " \
        f"{float(((got - ref).abs() / bound.clamp(min=1e-300)).nan_to_num(1e30).max()):.3g}"


# ------------------------------------------------------------------------------------------------------- norm + rotation
def _axis_of(dims):
    return torch.cat([torch.full((n,), a) for a, n in enumerate(dims)])


def _angles(pos, dims, base=10000.0):
    """pos [B, L, A] -> [B, L, columns] in 64 bits"""
    out = []
    for a, n in enumerate(dims):
        f = base ** (-torch.arange(n, dtype=torch.float64) / n)
        out.append(pos[..., a:a + 1].double() * f)
    return torch.cat(out, -1)


def _turn(y, ang, inter, back=False):
    half = ang.shape[-1]
    c, s = ang.cos().unsqueeze(2), ang.sin().unsqueeze(2) * (-1 if back else 1)
    z = y.clone()
    if inter:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        z[..., 0:2 * half:2], z[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        z[..., :half], z[..., half:2 * half] = a * c - b * s, b * c + a * s
    return z


def _norm_ref(x, w, ang, eps, inter):
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    return _turn(y, ang, inter) if ang is not None else y


def _norm_ref_backward(x, w, dz, ang, eps, inter):
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    dy = _turn(dz, ang, inter, back=True) if ang is not None else dz
    g = dy * w
    return r * (g - n * (g * n).mean(-1, keepdim=True)), dy * n


def _pair_abs(y, half, inter):
    """|a| + |b| of a column's pair, which a turned value is a combination of"""
    a = y.abs()
    if inter:
        s = a[..., 0:2 * half:2] + a[..., 1:2 * half:2]
        a = a.clone()
        a[..., 0:2 * half:2], a[..., 1:2 * half:2] = s, s
        return a
    s = a[..., :half] + a[..., half:2 * half]
    return torch.cat([s, s, a[..., 2 * half:]], -1)


# B, L, Hq, Hk, D, turned columns, axes (columns each), interleaved, fused projection, positions
NORM = [(1, 1, 1, 1, 24, 24, (12,), False, True, "row"),
        (2, 7, 3, 1, 32, 32, (6, 5, 5), False, True, "batch"),        # the columns of a load belong to two axes
        (1, 33, 2, 2, 64, 64, (32,), True, True, "batch"),
        (2, 5, 4, 2, 64, 32, (16,), False, False, None),              # half of the columns turned
        (1, 9, 1, 0, 128, 128, (64,), False, True, "row"),            # queries alone
        (3, 4, 5, 5, 6, 6, (3,), True, False, "batch"),
        (1, 6, 2, 1, 10, 4, (1, 1), False, False, "row"),
        (2, 3, 2, 2, 96, 0, None, False, True, None),                 # the norm alone
        (1, 70, 1, 1, 2, 2, (1,), False, False, None)]


def _norm_case(case, dtype, seed=3):
    B, L, Hq, Hk, D, rot, dims, inter, fused, kind = case
    n = (Hq + 2 * Hk) * D
    x = _randn((B, L, n), seed, 3.0).to(dtype)
    q, k = x[..., :Hq * D].unflatten(-1, (Hq, D)), None
    if Hk:
        k = x[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
    if not fused:
        q, k = q.contiguous(), None if k is None else k.contiguous()
    qw = (1 + _randn((D,), seed + 1, 0.2)).to(dtype)
    kw = (1 + _randn((D,), seed + 2, 0.2)).to(dtype) if Hk else None
    kws, ang = dict(eps=1e-5, interleaved=inter), None
    if rot:
        length = 4000
        cos, sin = rotary_table(length, rot, axis_dims=dims, device="cpu")
        kws.update(cos=cos, sin=sin, axis_dims=dims if len(dims) > 1 else None)
        if kind:
            shape = ((L,) if kind == "row" else (B, L)) + ((len(dims),) if len(dims) > 1 else ())
            pos = torch.randint(0, length, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
            kws["positions"] = pos
            full = pos.reshape((1 if kind == "row" else B), L, len(dims)).expand(B, L, len(dims))
        else:
            full = torch.arange(L)[None, :, None].expand(B, L, 1)
        ang = _angles(full, dims)
    return q, k, qw, kw, kws, ang


def _dev(be, kws):
    return {n: be.to(v) for n, v in kws.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", NORM)
def test_qk_norm_rope(be, case, dtype):
    D, rot, inter = case[4], case[5], case[7]
    q, k, qw, kw, kws, ang = _norm_case(case, dtype)
    qo, ko = be.ops.qk_norm_rope(*be.to(q, k, qw, kw), **_dev(be, kws))
    assert (ko is None) == (k is None)
    for name, x, w, z in (("q", q, qw, qo), ("k", k, kw, ko)):
        if x is None:
            continue
        assert z.is_contiguous() and z.dtype == dtype
        xd, wd = x.double(), w.double()
        ref = _norm_ref(xd, wd, ang, kws["eps"], inter)
        y = _norm_ref(xd, wd, None, kws["eps"], inter)
        # the mean of D squares, its root and quotient, two products, two products with table values rounded once, a sum
        mag = _pair_abs(y, rot // 2, inter) if rot else y.abs()
        _within(z, ref, (D / 2 + 16) * U * mag + _half(dtype) * ref.abs() + 1e-30, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", NORM)
def test_qk_norm_rope_backward(be, case, dtype):
    B, L, Hq, Hk, D, rot, _, inter, _, _ = case
    q, k, qw, kw, kws, ang = _norm_case(case, dtype)
    dq = _randn((B, L, Hq, D), 8).to(dtype)
    dk = _randn((B, L, Hk, D), 9).to(dtype) if Hk else None
    got = be.ops.qk_norm_rope_backward(*be.to(q, k, qw, kw, dq, dk), **_dev(be, kws))
    for name, x, w, dz, dx, dw in (("q", q, qw, dq, got[0], got[2]), ("k", k, kw, dk, got[1], got[3])):
        if x is None:
            assert dx is None and dw is None
            continue
        xd, wd, dzd = x.double(), w.double(), dz.double()
        ref, terms = _norm_ref_backward(xd, wd, dzd, ang, kws["eps"], inter)
        r = (xd.square().mean(-1, keepdim=True) + kws["eps"]).rsqrt()
        n = (xd * r).abs()
        g = (_pair_abs(dzd, rot // 2, inter) if rot else dzd.abs()) * wd.abs()
        mag = r * (g + n * (g * n).mean(-1, keepdim=True))
        _within(dx, ref, (2 * D + 32) * U * mag + _half(dtype) * ref.abs() + 1e-30, "d" + name)
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        total = terms.sum((0, 1, 2))
        tmag = (n * g / wd.abs()).sum((0, 1, 2))
        _within(dw, total, (rows + D + 32) * U * tmag + _half(dtype) * total.abs() + 1e-30, "dw" + name)


def test_gradients_by_differences():
    """the 64-bit formulas that the kernels are held to, against central differences of their forwards"""
    q, _, qw, _, kws, ang = _norm_case(NORM[5], torch.float32)
    x, w, dz = q.double().requires_grad_(), qw.double().requires_grad_(), _randn(q.shape, 1).double()
    f = lambda a, b: _norm_ref(a, b, ang, 1e-5, True)
    assert torch.autograd.gradcheck(f, (x, w))
    dx, dw = torch.autograd.grad(f(x, w), (x, w), dz)
    got, terms = _norm_ref_backward(x.detach(), w.detach(), dz, ang, 1e-5, True)
    assert torch.allclose(got, dx, atol=1e-12) and torch.allclose(terms.sum((0, 1, 2)), dw, atol=1e-12)

    case = (1, 5, 7, 2, 1, 8, True, 4, 3, False, [(5, 7, 2)])
    q, k, v, table, plan, lens, dout = _attn_inputs(case, torch.float32)

    def attend(q, k, v, table):
        rel = torch.arange(7)[None] - (2 + torch.arange(5))[:, None]
        t = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(2, 2)) * 8 ** -0.5 + table[plan.bucket(rel)].permute(2, 0, 1)
        return torch.einsum("bhij,bjhd->bihd", t.masked_fill(rel > 0, -math.inf).softmax(-1), v.repeat_interleave(2, 2))
    xs = tuple(t.double().requires_grad_() for t in (q, k, v, table))
    assert torch.autograd.gradcheck(attend, xs)
    want = torch.autograd.grad(attend(*xs), xs, dout.double())
    ref = _attn_ref(q, k, v, table, plan, True, 8 ** -0.5, *lens, dout, torch.float32)
    assert torch.allclose(ref["out"][0], attend(*xs), atol=1e-12)
    for name, g in zip(("dq", "dk", "dv", "dtable"), want):
        assert torch.allclose(ref[name][0], g, atol=1e-12), name


def test_qk_norm_rope_odd_addresses(be):
    """rows and tables that no wide load can read, and a row of zeros"""
    D = 24
    flat = _randn((2 * 3 * 2 * (D + 1) + 1,), 5)
    q = flat[1:].as_strided((2, 3, 2, D), (3 * 2 * (D + 1), 2 * (D + 1), D + 1, 1))
    q[0, 1, 0] = 0.0
    w = _randn((D + 1,), 6)[1:]
    cos, sin = rotary_table(8, D, device="cpu")
    for inter in (False, True):
        qo, _ = be.ops.qk_norm_rope(be.to(flat)[1:].as_strided(q.shape, q.stride()), None, be.to(_randn((D + 1,), 6))[1:], None,
                                    *be.to(cos, sin), interleaved=inter)
        ang = _angles(torch.arange(3)[None, :, None].expand(2, 3, 1), (D // 2,))
        ref = _norm_ref(q.double(), w.double(), ang, 1e-6, inter)
        y = _norm_ref(q.double(), w.double(), None, 1e-6, inter)
        _within(qo, ref, (D / 2 + 16) * U * _pair_abs(y, D // 2, inter) + 1e-30, "q")
        assert bool((qo[0, 1, 0] == 0).all())


def test_qk_norm_rope_far_positions_and_bounds(be):
    cos, sin = rotary_table(1_000_001, 4, device="cpu")
    q = _randn((1, 4, 1, 4), 2)
    pos = torch.tensor([1_000_000, 1_000_001, -1, 0], dtype=torch.int32)
    qo, _ = be.ops.qk_norm_rope(be.to(q), None, be.to(torch.ones(4)), None, *be.to(cos, sin, pos))
    qo = qo.cpu()
    assert bool(qo[0, 1:3].isnan().all()), "positions outside the table have to show"
    ref = _norm_ref(q.double(), torch.ones(4).double(), _angles(pos.clamp(0, 1_000_000)[None, :, None], (2,)), 1e-6, False)
    # 4 columns: the general bound of test_qk_norm_rope with the pairs' magnitudes taken as twice the row's largest
    _within(qo[:, ::3], ref[:, ::3], (20 * U * ref.abs().amax(-1, keepdim=True) * 2)[:, ::3], "q")


def test_qk_norm_rope_refusals(be):
    o = be.ops
    cos, sin = be.to(*rotary_table(8, 8, device="cpu"))
    q, w = be.to(_randn((1, 4, 2, 8), 1), torch.ones(8))
    bad = [dict(q=q[0]), dict(q=q.double()), dict(qw=w[:4]), dict(qw=w.bfloat16()), dict(k=q), dict(kw=w),
           dict(k=q[:, :3], kw=w), dict(k=q.bfloat16(), kw=w), dict(cos=None), dict(sin=None), dict(cos=cos[:4]),
           dict(cos=cos.bfloat16(), sin=sin.bfloat16()), dict(positions=torch.zeros(4, dtype=torch.int64, device=q.device)),
           dict(positions=torch.zeros(3, dtype=torch.int32, device=q.device)), dict(axis_dims=(2, 1)), dict(axis_dims=(2, 2)),
           dict(q=q[:, :0]), dict(q=q.expand(1, 4, 2, 8)[..., :7], qw=w[:7], cos=None, sin=None)]
    for b in bad:
        a = dict(q=q, k=None, qw=w, kw=None, cos=cos, sin=sin, positions=None, axis_dims=None)
        a.update(b)
        with pytest.raises(OccfError):
            o.qk_norm_rope(a["q"], a["k"], a["qw"], a["kw"], a["cos"], a["sin"], a["positions"], axis_dims=a["axis_dims"])
    with pytest.raises(OccfError):
        o.qk_norm_rope_backward(q, None, w, None, q[:, :2], None, cos, sin)
    with pytest.raises(OccfError):
        o.qk_norm_rope_backward(q, q, w, w, q, None, cos, sin)
    for kw in (dict(rot_dim=7), dict(rot_dim=8, axis_dims=(1, 2)), dict(rot_dim=8, length=0), dict(rot_dim=8, axis_dims=(1, 1, 1, 1))):
        with pytest.raises(ValueError):
            rotary_table(**{"length": 4, "device": "cpu", **kw})


# ------------------------------------------------------------------------------------------------------- buckets
@pytest.mark.parametrize("n,R,both", [(32, 128, True), (32, 128, False), (8, 40, True), (4, 9, False), (64, 500, True), (2, 5, False)])
def test_relative_buckets(n, R, both):
    """every distance by the definition, in whole numbers"""
    t = RelativeBuckets(n, R, both, device="cpu")
    side = n // 2 if both else n
    e = side // 2
    for d in range(-R - 3, R + 4):
        a = abs(d) if both else max(0, -d)
        b = a if a < e else e + max(m for m in range(side - e) if min(a, R) ** (side - e) >= e ** (side - e - m) * R ** m)
        want = b + (side if both and d > 0 else 0)
        assert int(t.bucket(torch.tensor([d]))) == want, d
    assert int(t.lut.max()) < n and t.lut.numel() == 2 * R + 1


def test_relative_buckets_refusals():
    for kw in (dict(num_buckets=3), dict(num_buckets=130), dict(num_buckets=2), dict(max_distance=8), dict(max_distance=513),
               dict(num_buckets=1, bidirectional=False)):
        with pytest.raises(ValueError):
            RelativeBuckets(**{"device": "cpu", **kw})


# ------------------------------------------------------------------------------------------------------- attention
def _attn_ref(q, k, v, table, plan, causal, scale, q_lens, k_lens, q_start, dout, dtype):
    """64-bit forward and backward and the bounds of their errors.  -> {name: (value, bound)}"""
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    bf = BF if dtype == torch.bfloat16 else 0.0                 # rounding of P and dS before a product
    fin = _half(dtype)
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64)
    out = {n: [z(t), z(t)] for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v), ("dtable", table))}
    out["lse"] = [torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64), torch.zeros(B, Hq, Lq, dtype=torch.float64)]
    for b in range(B):
        n, m, s0 = int(q_lens[b]), int(k_lens[b]), int(q_start[b])
        if not n or not m:
            continue
        rel = torch.arange(m)[None] - (s0 + torch.arange(n))[:, None]
        bucket = plan.bucket(rel)
        for h in range(Hq):
            Q, K, V = q[b, :n, h].double(), k[b, :m, h // G].double(), v[b, :m, h // G].double()
            bias = table[:, h].double()[bucket]
            t = Q @ K.t() * scale + bias
            hide = (bias <= -1e30) | ((rel > 0) if causal else torch.zeros_like(rel, dtype=torch.bool))
            t = t.masked_fill(hide, -math.inf)
            some = ~hide.all(-1)
            P = torch.softmax(t, -1).nan_to_num(0.0)
            # a score: D products of values exact to 2^-22, their sum, scale and bias in base 2; then the difference to the
            # maximum; exp2 one step more.  Relative error of an unnormalised probability, and of P after the sum of m of them
            tmag = (Q.abs() @ K.abs().t() * scale).amax() + bias.masked_fill(hide, 0).abs().amax()
            lmag = t.masked_fill(hide, 0).abs().amax() + math.log(m)
            ep = float(((D + 12) * tmag + 6 * lmag + 2 * m + 16) * U)
            o = P @ V
            eo = (2 * ep + m * U + bf) * (P @ V.abs()) + fin * o.abs()
            out["out"][0][b, :n, h], out["out"][1][b, :n, h] = o, eo
            lse = torch.logsumexp(t, -1) / math.log(2)
            out["lse"][0][b, h, :n] = torch.where(some, lse, -math.inf)
            out["lse"][1][b, h, :n] = ep * 2 + 4 * U * lse.abs().nan_to_num(0, 0, 0)
            if dout is None:
                continue
            dO = dout[b, :n, h].double()
            dP = dO @ V.t()
            delta = (dO * o).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            edelta = (dO.abs() * eo).sum(-1, keepdim=True) + (D + 4) * U * (dO.abs() * o.abs()).sum(-1, keepdim=True)
            edP = (D + 12) * U * (dO.abs() @ V.abs().t())
            eS = 2 * ep * dS.abs() + P * (edP + edelta)
            eSr = eS + bf * dS.abs()
            out["dv"][0][b, :m, h // G] += P.t() @ dO
            out["dv"][1][b, :m, h // G] += (2 * ep + bf + n * U) * (P.t() @ dO.abs())
            out["dq"][0][b, :n, h] = scale * dS @ K
            out["dq"][1][b, :n, h] = scale * (eSr @ K.abs() + m * U * (dS.abs() @ K.abs()))
            out["dk"][0][b, :m, h // G] += scale * dS.t() @ Q
            out["dk"][1][b, :m, h // G] += scale * (eSr.t() @ Q.abs() + n * G * U * (dS.abs().t() @ Q.abs()))
            one = torch.nn.functional.one_hot(bucket.flatten().long(), plan.num_buckets).double()
            out["dtable"][0][:, h] += dS.flatten() @ one
            out["dtable"][1][:, h] += (eS + (n + m) * U * dS.abs()).flatten() @ one
    for name in ("dq", "dk", "dv", "dtable"):
        out[name][1] += (fin + 4 * U) * out[name][0].abs() + 1e-30
    out["out"][1] += 1e-30
    return out


# B, Lq, Lk, Hq, Hk, D, causal, buckets, radius, both sides, rows (queries, keys, position of the first query) a sequence
ATTN = [(1, 1, 1, 1, 1, 8, False, 8, 5, True, None),
        (1, 33, 33, 1, 1, 24, False, 8, 9, True, None),
        (2, 70, 70, 2, 1, 32, True, 8, 20, False, [(70, 70, 0), (37, 37, 0)]),
        (2, 40, 130, 2, 2, 64, True, 16, 16, False, [(40, 130, 90), (7, 65, 58)]),
        (3, 60, 60, 1, 1, 16, False, 8, 9, True, [(60, 60, 0), (0, 0, 0), (33, 1, 0)]),          # an empty sequence
        (1, 35, 40, 1, 1, 96, True, 8, 20, False, [(35, 40, -5)]),                               # queries before every key
        (1, 129, 65, 1, 1, 128, False, 8, 40, True, None)]


def _attn_inputs(case, dtype, seed=11):
    B, Lq, Lk, Hq, Hk, D, causal, nb, R, both, rows = case
    rows = rows or [(Lq, Lk, 0)] * B
    kv = _randn((B, Lk, 2 * Hk * D), seed).to(dtype)                     # keys and values as blocks of one projection
    q, dout = _randn((B, Lq, Hq, D), seed + 1, 1.5).to(dtype), _randn((B, Lq, Hq, D), seed + 2).to(dtype)
    for b, (n, m, _) in enumerate(rows):                                 # what does not count is never looked at
        q[b, n:], dout[b, n:], kv[b, m:] = NAN, NAN, NAN
    k, v = (kv[..., i * Hk * D:(i + 1) * Hk * D].unflatten(-1, (Hk, D)) for i in (0, 1))
    table = _randn((nb, Hq), seed + 3).to(dtype)
    plan = RelativeBuckets(nb, R, both, device="cpu")
    lens = [torch.tensor([r[i] for r in rows], dtype=torch.int32) for i in range(3)]
    return q, k, v, table, plan, lens, dout


def _plan_on(be, plan):
    return RelativeBuckets(plan.num_buckets, plan.radius, plan.bidirectional, device=be.device)


def _check_attention(be, case, dtype, backward=True, seed=11):
    causal = case[6]
    q, k, v, table, plan, lens, dout = _attn_inputs(case, dtype, seed)
    scale = case[5] ** -0.5
    ref = _attn_ref(q, k, v, table, plan, causal, scale, *lens, dout if backward else None, dtype)
    kw = dict(causal=causal)
    if case[10] is not None:
        kw.update(q_lens=be.to(lens[0]), k_lens=be.to(lens[1]), q_start=be.to(lens[2]))
    dq, dk, dv, dplan = be.to(q), be.to(k), be.to(v), _plan_on(be, plan)
    out, lse = be.ops.rel_attention(dq, dk, dv, be.to(table), dplan, return_lse=True, **kw)
    _within(out, *ref["out"], "out")
    finite = ref["lse"][0] > -math.inf
    assert torch.equal(lse.cpu() > -math.inf, finite)
    _within(lse.cpu()[finite], ref["lse"][0][finite], ref["lse"][1][finite], "lse")
    alone = be.ops.rel_attention(dq, dk, dv, be.to(table), dplan, **kw)
    assert torch.equal(alone, out)
    if not backward:
        return
    got = be.ops.rel_attention_backward(dq, dk, dv, be.to(table), dplan, out, lse, be.to(dout), **kw)
    for name, g in zip(("dq", "dk", "dv", "dtable"), got):
        assert g.dtype == dtype
        _within(g, *ref[name], name)
    for b, (n, m, _) in enumerate(case[10] or []):
        assert bool((got[0][b, n:] == 0).all()) and bool((got[1][b, m:] == 0).all()) and bool((got[2][b, m:] == 0).all())
    again = be.ops.rel_attention_backward(dq, dk, dv, be.to(table), dplan, out, lse, be.to(dout), **kw)
    assert all(torch.equal(a, g) for a, g in zip(again, got)), "two runs differ"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", ATTN)
def test_rel_attention(be, case, dtype):
    _check_attention(be, case, dtype)


# walks longer than 512: the bf16 backward rounds P and dS once instead of taking two pieces
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 3, 515, 2, 1, 24, True, 8, 20, False, [(3, 515, 512)]),
                                  (2, 520, 33, 1, 1, 64, False, 8, 9, True, [(520, 33, 0), (77, 1, -40)]),
                                  (1, 5, 513, 1, 1, 96, False, 8, 40, True, None),
                                  (1, 514, 2, 1, 1, 128, True, 8, 9, False, [(513, 2, 0)])])
def test_rel_attention_long_walks(be, case, dtype):
    _check_attention(be, case, dtype)


@pytest.mark.parametrize("case", [(1, 55, 55, 2, 2, 32, False, 32, 40, True, None), (2, 40, 11, 4, 2, 24, True, 8, 40, False, None),
                                  (1, 94, 94, 4, 2, 64, True, 16, 40, True, None)])
def test_rel_attention_short_walks_round_once(be, case):
    """bf16 gradients of short walks: no further off, in the mean square, than their own last rounding of the exact value and a
    tenth (what else there is, 2^-16 of dS and P, would have to be 0.45 of it to show)"""
    q, k, v, table, plan, lens, dout = _attn_inputs(case, torch.bfloat16)
    ref = _attn_ref(q, k, v, table, plan, case[6], case[5] ** -0.5, *lens, dout, torch.bfloat16)
    dq, dk, dv, tb, do = be.to(q), be.to(k), be.to(v), be.to(table), be.to(dout)
    out, lse = be.ops.rel_attention(dq, dk, dv, tb, _plan_on(be, plan), causal=case[6], return_lse=True)
    got = be.ops.rel_attention_backward(dq, dk, dv, tb, _plan_on(be, plan), out, lse, do, causal=case[6])
    for name, g in zip(("dq", "dk", "dv", "dtable"), got):
        want = ref[name][0]
        assert float((g.cpu().double() - want).norm()) <= 1.1 * float((want.bfloat16().double() - want).norm()), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,causal", [(24, False), (64, True), (96, False), (128, True)])
def test_rel_attention_many_rows(be, D, causal, dtype):
    """enough rows that the kernel for many queries takes them: 130 heads of 40 queries and 70 keys, one sequence shorter than a
    tile, one empty, one whose queries stand before every key"""
    rows = [(40, 70, 30)] * 9 + [(33, 5, 0), (0, 0, 0), (40, 33, -20), (12, 70, 0)]
    _check_attention(be, (13, 40, 70, 10, 5, D, causal, 8, 12, not causal, rows), dtype, backward=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 36, 70, 344, 172, 24, False, 8, 12, True, [(33, 65, 0)]),
                                  (1, 36, 70, 176, 44, 64, True, 8, 12, False, [(36, 70, 34)])])
def test_rel_attention_many_heads(be, case, dtype):
    """enough heads of 32 and 64 columns that the kernel for many queries takes them"""
    _check_attention(be, case, dtype, backward=False)


@pytest.mark.parametrize("Lq", [260, 129])
def test_rel_attention_causal_tiles(be, Lq):
    """causal, several tiles of 128 queries and more heads than one round of the workgroups' order takes"""
    heads = 256
    case = (1, Lq, Lq, heads, heads // 8, 8, True, 8, 12, False, [(Lq, Lq - 5, 3)])
    q, k, v, table, plan, lens, _ = _attn_inputs(case, torch.bfloat16)
    ref = _attn_ref(q, k, v, table, plan, True, 8 ** -0.5, *lens, None, torch.bfloat16)
    out = be.ops.rel_attention(*be.to(q, k, v, table), _plan_on(be, plan), causal=True, q_lens=be.to(lens[0]),
                               k_lens=be.to(lens[1]), q_start=be.to(lens[2]))
    _within(out, *ref["out"], "out")


# key lengths of the sequences; None: all keys of all
SINGLE = [(2, 700, 1, 1, 32, None), (3, 700, 4, 2, 24, [700, 0, 129]), (5, 513, 17, 1, 64, [1, 127, 128, 513, 400]),
          (70, 300, 2, 2, 8, [(37 * b) % 301 for b in range(70)]), (2, 260, 32, 1, 128, [260, 31])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", SINGLE)
def test_rel_attention_single_queries(be, case, dtype):
    """one query a sequence against its keys so far: 16 and 32 rows a key head, walks cut by the longest sequence and by every
    sequence's own length, more sequences than a wave has lanes"""
    B, Lk, G, Hk, D, lens = case
    n = lens or [Lk] * B
    rows = [(1, m, m - 1) for m in n]
    _check_attention(be, (B, 1, Lk, G * Hk, Hk, D, True, 8, 40, False, rows), dtype, backward=False)
    if lens is None:
        q, k, v, table, plan, (_, _, start), _ = _attn_inputs((B, 1, Lk, G * Hk, Hk, D, True, 8, 40, False, rows), dtype)
        a = be.to(q, k, v, table)
        want = be.ops.rel_attention(*a, _plan_on(be, plan), causal=True, q_start=be.to(start))
        lens = be.to(torch.tensor(n, dtype=torch.int32))
        got = be.ops.rel_attention(*a, _plan_on(be, plan), causal=True, q_start=be.to(start), k_lens=lens)
        # the same keys in other parts: as in test_prompt_then_single_tokens
        tol = (3 * BF if dtype == torch.bfloat16 else (4 * Lk + 8 * D) * U) * float(v.abs().amax())
        assert float((want - got).abs().max()) <= tol


# keys in several parts, of either type
LONG_SINGLE = [(2, 1030, 1, 1, 32, None), (3, 1100, 4, 2, 24, [1100, 0, 129]), (5, 1030, 17, 1, 64, [1, 127, 128, 1030, 400]),
               (70, 1030, 2, 1, 8, [(37 * b) % 1031 for b in range(70)]), (2, 2060, 32, 1, 128, [260, 2060]),
               (3, 1700, 4, 2, 24, [1700, 0, 129]), (70, 1540, 2, 1, 8, [(37 * b) % 1541 for b in range(70)])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", LONG_SINGLE)
def test_rel_attention_single_queries_long(be, case, dtype):
    """by parts of the keys: the wave that joins them, parts by the sequences' lengths, sequences of none"""
    test_rel_attention_single_queries(be, case, dtype)


def test_rel_attention_lengths_out_of_range(be):
    """lengths beyond the tensors count as all of it, negative ones as none; positions far outside stay far outside"""
    q, k, v, table, plan, _, dout = _attn_inputs((4, 40, 40, 2, 2, 32, False, 8, 9, True, None), torch.float32)
    i32 = lambda *x: be.to(torch.tensor(x, dtype=torch.int32))
    a = [*be.to(q, k, v, table), _plan_on(be, plan)]
    big = 2 ** 31 - 1
    for (ql, kl, st), (ql2, kl2, st2) in ((((41, big, -1, 40), (big, 41, 40, -big), (0,) * 4), ((40, 40, 0, 40), (40, 40, 40, 0), (0,) * 4)),
                                          (((40,) * 4, (40,) * 4, (big, -big, 1 << 30, -(1 << 30))),
                                           ((40,) * 4, (40,) * 4, (1 << 20, -(1 << 20), 1 << 20, -(1 << 20))))):
        r = [be.ops.rel_attention(*a, q_lens=i32(*x), k_lens=i32(*y), q_start=i32(*z), return_lse=True)
             for x, y, z in ((ql, kl, st), (ql2, kl2, st2))]
        assert torch.equal(r[0][0], r[1][0]) and torch.equal(r[0][1], r[1][1])
        g = [be.ops.rel_attention_backward(*a, *o, be.to(dout), q_lens=i32(*x), k_lens=i32(*y), q_start=i32(*z))
             for o, (x, y, z) in zip(r, ((ql, kl, st), (ql2, kl2, st2)))]
        assert all(torch.equal(x, y) for x, y in zip(*g))


def test_rel_attention_taken_out_buckets(be):
    """a table entry at the type's lowest value or -inf takes its bucket out, and a row left with nothing is zeros"""
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, table, plan, lens, dout = _attn_inputs((1, 40, 40, 2, 2, 32, False, 8, 9, True, None), dtype)
        table[3, 0], table[7, 0], table[:, 1] = torch.finfo(dtype).min, -math.inf, -math.inf
        ref = _attn_ref(q, k, v, table, plan, False, 32 ** -0.5, *lens, dout, dtype)
        a = [be.to(t) for t in (q, k, v, table)] + [_plan_on(be, plan)]
        out, lse = be.ops.rel_attention(*a, return_lse=True)
        _within(out, *ref["out"], "out")
        assert bool((out[:, :, 1] == 0).all()) and bool((lse[:, 1] == -math.inf).all())
        for name, g in zip(("dq", "dk", "dv", "dtable"), be.ops.rel_attention_backward(*a, out, lse, be.to(dout))):
            _within(g, *ref[name], name)


def test_rel_attention_strides_and_addresses(be):
    """head-major tensors, rows off 16-byte addresses and column strides other than 1 give what contiguous tensors give"""
    q, k, v, table, plan, _, dout = _attn_inputs((2, 20, 33, 4, 2, 24, False, 8, 9, True, None), torch.float32)
    plan = _plan_on(be, plan)
    a = [be.to(t.contiguous()) for t in (q, k, v)]
    table, dout = be.to(table), be.to(dout)
    want, lse = be.ops.rel_attention(*a, table, plan, return_lse=True)
    grads = be.ops.rel_attention_backward(*a, table, plan, want, lse, dout)

    def head_major(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def off(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    def columns(t):
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    for f in (head_major, off, columns):
        b = [f(t) for t in a]
        assert torch.equal(be.ops.rel_attention(*b, off(table), plan), want)
        for x, y in zip(be.ops.rel_attention_backward(*b, table, plan, f(want), lse, f(dout)), grads):
            assert torch.equal(x, y)
    one = a[0][:, :1].expand(2, 20, 4, 24)                               # a query row repeated: row stride 0
    assert torch.equal(be.ops.rel_attention(one, a[1], a[2], table, plan), be.ops.rel_attention(one.contiguous(), a[1], a[2], table, plan))


def test_rel_attention_refusals(be):
    q, k, v, table, plan, lens, dout = _attn_inputs((2, 8, 9, 4, 2, 16, False, 8, 9, True, None), torch.float32)
    q, k, v, table, dout, plan = *be.to(q, k, v, table, dout), _plan_on(be, plan)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=q.device)
    bad = [dict(q=q[0]), dict(q=q.double()), dict(q=q.bfloat16()), dict(q=q[:, :0]), dict(k=k[:, :, :, :8]), dict(k=k[:1], v=v[:1]),
           dict(v=v[:, :5]), dict(k=k[:, :, :1].expand(2, 9, 3, 16), v=v[:, :, :1].expand(2, 9, 3, 16)), dict(table=table[:4]),
           dict(table=table[:, :2]), dict(table=table.bfloat16()), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
           dict(scale=NAN), dict(q_lens=i32(1)), dict(k_lens=i32(1, 2).long()), dict(q_start=i32(1, 2, 3)),
           dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), dict(k=k[:, :0], v=v[:, :0])]
    for b in bad:
        a = dict(q=q, k=k, v=v, table=table, buckets=plan)
        a.update(b)
        with pytest.raises(OccfError):
            be.ops.rel_attention(**a)
    wide = [t.repeat(1, 1, 1, 9) for t in (q, k, v)]                     # 144 columns
    with pytest.raises(OccfError):
        be.ops.rel_attention(*wide, table, plan)
    out, lse = be.ops.rel_attention(q, k, v, table, plan, return_lse=True)
    for o, l, d in ((out[:, :4], lse, dout), (out, lse[:1], dout), (out, lse.double(), dout), (out, lse, dout.bfloat16()),
                    (out, lse, dout[..., :8])):
        with pytest.raises(OccfError):
            be.ops.rel_attention_backward(q, k, v, table, plan, o, l, d)


def test_rel_attention_c_entry_refuses(be):
    """the C entry checks what it is given by itself: nothing is launched"""
    import ctypes
    lib, n = be.ops.lib, ctypes.c_void_p(0)
    good = [1, 4, 4, 2, 2, 16, 8, 9] + [128, 32, 16] * 3
    for at, value in ((0, 0), (1, 0), (2, -1), (3, 3), (4, 0), (5, 12), (5, 136), (6, 129), (6, 0), (7, 0), (7, 513), (8, 6), (12, 3)):
        g = list(good)
        g[at] = value
        assert lib.occf_rel_attn_workspace((ctypes.c_int64 * 17)(*g), 1) == -1
        assert lib.occf_rel_attn_bwd_workspace((ctypes.c_int64 * 17)(*g), 0, 1) == -1
    g = (ctypes.c_int64 * 17)(*good)
    assert lib.occf_rel_attn_workspace(g, 2) == -1 and lib.occf_rel_attn_workspace(g, 0) >= 0
    assert lib.occf_rel_attn_fwd(n, n, n, n, n, n, n, n, n, n, n, 0, g, 1.0, 0, 0, n) < 0
    assert lib.occf_rel_attn_bwd(*[n] * 16, 0, g, 1.0, 0, 0, n) < 0
    g = (ctypes.c_int64 * 17)(1, 4, 2, 0, 8, 8, 4, 1, 4, 4, 0, 64, 16, 8, 0, 0, 0)
    assert lib.occf_qk_norm_rope_fwd(*[n] * 9, g, 1e-6, 0, 0, n) < 0
    assert lib.occf_qk_norm_rope_bwd(*[n] * 14, g, 1e-6, 0, 0, n) < 0


def test_qk_norm_rope_c_entry_refuses_axes(be):
    """two axes whose columns do not fill the table would read a third coordinate that the positions do not have"""
    import ctypes
    q, w = be.to(_randn((1, 4, 2, 8), 1), torch.ones(8))
    cos, sin = be.to(*rotary_table(8, 8, device="cpu"))
    pos, out = be.to(torch.zeros((4, 2), dtype=torch.int32)), torch.empty_like(q)
    for axes, cuts in ((2, (2, 3)), (2, (3, 2)), (2, (0, 4)), (3, (0, 2))):
        g = (ctypes.c_int64 * 17)(1, 4, 2, 0, 8, 8, 8, axes, *cuts, 0, 64, 16, 8, 0, 0, 0)
        ptr = [t if t is None else t.data_ptr() for t in (q, None, w, None, cos, sin, pos, out, None)]
        assert be.ops.lib.occf_qk_norm_rope_fwd(*ptr, g, 1e-6, 0, 0, ctypes.c_void_p(0)) < 0
        ptr = [t if t is None else t.data_ptr() for t in (q, None, w, None, cos, sin, pos, out, None, out, None, w, None, out)]
        assert be.ops.lib.occf_qk_norm_rope_bwd(*ptr, g, 1e-6, 0, 0, ctypes.c_void_p(0)) < 0


def _step(ops, x, w, table, plan, cos, sin, pos, lens, Hq, Hk, D, causal):
    q, k, v = x.split((Hq * D, Hk * D, Hk * D), -1)
    heads = lambda t: t.unflatten(-1, (-1, D))
    q, k = ops.qk_norm_rope(heads(q), heads(k), w[0], w[1], cos, sin, pos)
    return q, k, heads(v), ops.rel_attention(q, k, heads(v), table, plan, causal=causal, q_lens=lens, k_lens=lens, return_lse=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_single_tokens(be, dtype):
    """as they are used together: a projection's rows are normed, turned and attended in one go; the same rows one by one against
    the keys kept so far give the same outputs"""
    B, L, Hq, Hk, D = 2, 37, 4, 2, 32
    x = _randn((B, L, (Hq + 2 * Hk) * D), 21).to(dtype)
    w = [(1 + _randn((D,), s, 0.1)).to(dtype) for s in (1, 2)]
    table = _randn((8, Hq), 3).to(dtype)
    plan = RelativeBuckets(8, 12, False, device=be.device)
    cos, sin = rotary_table(64, D, device=be.device)
    x, w, table = be.to(x), be.to(*w), be.to(table)
    lens = be.to(torch.tensor([L, L], dtype=torch.int32))
    q, k, v, (out, _) = _step(be.ops, x, w, table, plan, cos, sin, None, lens, Hq, Hk, D, True)
    kept_k, kept_v = (torch.full((B, 48, Hk, D), NAN, dtype=dtype, device=x.device) for _ in range(2))
    for i in range(L):
        at = torch.full((B, 1), i, dtype=torch.int32, device=x.device)
        xi = x[:, i:i + 1]
        qi, ki, vi = xi.split((Hq * D, Hk * D, Hk * D), -1)
        qi, ki = be.ops.qk_norm_rope(qi.unflatten(-1, (Hq, D)), ki.unflatten(-1, (Hk, D)), *w, cos, sin, at)
        assert torch.equal(qi[:, 0], q[:, i]) and torch.equal(ki[:, 0], k[:, i])
        kept_k[:, i], kept_v[:, i] = ki[:, 0], vi.unflatten(-1, (Hk, D))[:, 0]
        oi = be.ops.rel_attention(qi, kept_k, kept_v, table, plan, causal=True, k_lens=at[:, 0] + 1, q_start=at[:, 0].contiguous())
        # the same keys in other tiles: sums of up to L + D terms in another order, and bf16 once more on P and the output
        tol = (3 * BF if dtype == torch.bfloat16 else (4 * L + 8 * D) * U) * float(v.abs().amax())
        assert float((oi[:, 0] - out[:, i]).abs().max()) <= tol


def test_training_step_through_autograd(be, monkeypatch):
    """norm, rotation and attention in one graph; every gradient against the 64-bit graph"""
    from occformer_amd import autograd as A
    monkeypatch.setattr(A, "get_ops", lambda: be.ops)
    B, L, H, D = 2, 40, 2, 32
    x = _randn((B, L, 3 * H * D), 31)
    w = [1 + _randn((D,), s, 0.1) for s in (1, 2)]
    table, dout = _randn((8, H), 3), _randn((B, L, H, D), 4)
    plan = RelativeBuckets(8, 9, True, device=be.device)
    cos, sin = rotary_table(64, D, device="cpu")
    lens = torch.tensor([40, 23], dtype=torch.int32)
    dout[1, 23:] = 0

    def graph(x, w0, w1, table):
        q, k, v = (t.unflatten(-1, (H, D)) for t in x.chunk(3, -1))
        ang = _angles(torch.arange(L)[None, :, None].expand(B, L, 1), (D // 2,))
        q, k = _norm_ref(q, w0, ang, 1e-6, False), _norm_ref(k, w1, ang, 1e-6, False)
        rel = torch.arange(L)[None] - torch.arange(L)[:, None]
        cpu = RelativeBuckets(8, 9, True, device="cpu")
        t = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5 + table[cpu.bucket(rel)].permute(2, 0, 1)
        t = t.masked_fill(torch.arange(L) >= lens[:, None, None, None], -math.inf)
        return torch.einsum("bhij,bjhd->bihd", t.softmax(-1), v)
    ref_in = [t.double().requires_grad_() for t in (x, *w, table)]
    ref = graph(*ref_in)
    want = torch.autograd.grad(ref, ref_in, dout.double())
    leaves = [be.to(t).requires_grad_() for t in (x, *w, table)]
    q, k, v = (t.unflatten(-1, (H, D)) for t in leaves[0].chunk(3, -1))
    q, k = A.qk_norm_rope(q, k, leaves[1], leaves[2], *be.to(cos, sin))
    out = A.rel_attention(q, k, v, leaves[3], plan, q_lens=be.to(lens), k_lens=be.to(lens))
    got = torch.autograd.grad(out, leaves, be.to(dout))
    # sums of L, D and B H L^2 products whose factors carry about (D + L) u each; magnitudes up to the largest gradient
    for g, r in zip(got, want):
        assert float((g.cpu().double() - r).norm() / r.norm()) <= 8 * (D + L) * U


# ------------------------------------------------------------------------------------------------------- on the device
@pytest.mark.gpu
@pytest.mark.parametrize("case", [(2, 500, 500, 8, 2, 128, True, 32, 128, False, [(500, 500, 0), (333, 333, 0)]),
                                  (1, 1100, 1100, 4, 4, 24, False, 32, 300, True, None),
                                  (4, 1030, 1030, 32, 32, 64, True, 32, 128, False, None),     # more workgroups than walks to cut
                                  (1, 300, 2000, 6, 2, 96, True, 16, 500, False, [(300, 2000, 1700)])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rel_attention_larger(hip, case, dtype):
    _check_attention(hip, case, dtype)


@pytest.mark.gpu
def test_rel_attention_far_offsets(hip):
    """keys beyond 2^31 elements from the first, across a batch and along one sequence's rows"""
    D, L = 64, 1 << 15
    q, table = hip.to(_randn((2, 1, 1, D), 1).bfloat16()), hip.to(_randn((8, 1), 2).bfloat16())
    plan = RelativeBuckets(8, 40, False, device=hip.device)
    kv = hip.to(_randn((2, L, 2, D), 3).bfloat16())
    lens = hip.to(torch.tensor([L, L - 77], dtype=torch.int32))
    want = hip.ops.rel_attention(q, kv[:, :, :1], kv[:, :, 1:], table, plan, causal=True, k_lens=lens, q_start=lens - 1)
    for shape, stride in (((2, L, 2, D), (1 << 31, 2 * D, D, 1)), ((2, L, 2, D), (2 * D, 1 << 17, D, 1))):
        flat = torch.zeros(((shape[0] - 1) * stride[0] + shape[1] * stride[1],), dtype=torch.bfloat16, device=hip.device)
        far = flat.as_strided(shape, stride)
        far.copy_(kv)
        got = hip.ops.rel_attention(q, far[:, :, :1], far[:, :, 1:], table, plan, causal=True, k_lens=lens, q_start=lens - 1)
        assert torch.equal(got, want)
        del flat, far


@pytest.mark.gpu
def test_position_operators_in_a_graph_and_on_a_stream(hip):
    """forward and backward captured twice and replayed in turn between eager calls on other inputs, and everything on a stream
    of its own (no eager graph of the leaves is alive during a capture: torch does not allow that)"""
    from occformer_amd import autograd as A
    B, L, H, D = 2, 200, 4, 64
    plan = RelativeBuckets(32, 64, True, device=hip.device)
    cos, sin = rotary_table(256, D)
    lens = hip.to(torch.tensor([200, 131], dtype=torch.int32))
    leaves = [hip.to(_randn(s, i)).bfloat16().requires_grad_() for i, s in enumerate([(B, L, 3 * H * D), (D,), (D,), (32, H)])]
    dout = hip.to(_randn((B, L, H, D), 9)).bfloat16()

    def forward():
        q, k, v = (t.unflatten(-1, (H, D)) for t in leaves[0].chunk(3, -1))
        q, k = A.qk_norm_rope(q, k, leaves[1], leaves[2], cos, sin)
        return A.rel_attention(q, k, v, leaves[3], plan, q_lens=lens, k_lens=lens)

    def step():
        out = forward()
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for n in range(4):
        with torch.no_grad():
            leaves[0].copy_(hip.to(_randn((B, L, 3 * H * D), 50 + n)))
        want = step()
        torch.cuda.synchronize()
        for g, outs in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), n
        with torch.cuda.stream(side):
            other = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, want))


@pytest.mark.gpu
def test_position_operators_refuse_mixed_devices(hip):
    q, w = hip.to(_randn((1, 4, 2, 8), 1)), torch.ones(8)
    with pytest.raises(OccfError):
        hip.ops.qk_norm_rope(q, None, w, None)
    with pytest.raises(OccfError):
        hip.ops.qk_norm_rope(q.cpu(), None, w, None)
    plan = RelativeBuckets(8, 9, True, device="cpu")
    with pytest.raises(OccfError):
        hip.ops.rel_attention(q, q, q, hip.to(_randn((8, 2), 1)), plan)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [2, 16])
def test_rel_attention_far_rows_training(hip, H):
    """rows of queries, keys and values beyond 2^31 elements from the first, forward (both kernels) and backward: the same bits as
    from rows side by side"""
    L, D, step = 2100, 64, 1 << 20
    x = hip.to(_randn((1, L, 3, H, D), 41).bfloat16())
    table, dout = hip.to(_randn((8, H), 42).bfloat16()), hip.to(_randn((1, L, H, D), 43).bfloat16())
    plan = RelativeBuckets(8, 40, True, device=hip.device)
    flat = torch.zeros((L * step,), dtype=torch.bfloat16, device=hip.device)
    far = flat.as_strided((1, L, 3, H, D), (L * step, step, H * D, D, 1))
    far.copy_(x)
    got = []
    for t in (x, far):
        q, k, v = t.unbind(2)
        out, lse = hip.ops.rel_attention(q, k, v, table, plan, return_lse=True)
        got.append((out, lse, *hip.ops.rel_attention_backward(q, k, v, table, plan, out, lse, dout)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    w = torch.ones(D, device=hip.device).bfloat16()
    cos, sin = rotary_table(L, D, device=hip.device)
    a, b = ([*hip.ops.qk_norm_rope(t[:, :, 0], t[:, :, 1], w, w, cos, sin),
             *hip.ops.qk_norm_rope_backward(t[:, :, 0], t[:, :, 1], w, w, dout, dout, cos, sin)] for t in (x, far))
    for y, z in zip(a, b):
        assert torch.equal(y, z)
