"""Position operators where a value, a row or a layout is out of the ordinary: infinities and the largest numbers, rows and keys
that nothing reaches, long sums, refusals.  Definitions and bounds as in test_position_ops.py."""
import math

import pytest
import torch

from occformer_amd.position import RelativeBuckets
from tests.test_position_ops import NAN, U, _attn_inputs, _attn_ref, _check_attention, _plan_on, _randn, _within

# few queries; enough heads that the kernel for many queries takes the call (B, Lq, Lk, Hq, Hk, D, causal, buckets, radius, both
# sides, rows)
FEW = (1, 40, 40, 2, 2, 32, False, 8, 9, True, [(40, 39, 0)])
MANY = (1, 40, 40, 56, 28, 128, False, 8, 9, True, [(40, 39, 0)])


def _last_key_hidden(be, case, dtype, low):
    """a call whose last key is hidden by ``low`` in a column where every query is 1, and the reference without that key"""
    q, k, v, table, plan, lens, dout = _attn_inputs(case, dtype)
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[:, -1], v[:, -1] = 0.5, 2.0
    k[:, -1, :, 0] = low
    want = k.clone()
    want[:, -1] = 0.0
    return q, k, v, table, plan, dout, _attn_ref(q, want, v, table, plan, case[6], case[5] ** -0.5, *lens, dout, dtype)



@pytest.mark.parametrize("low", ["lowest", "-inf"])
def test_rel_attention_rows_behind_the_last_meet_an_infinite_key(be, low):
    """a mask as one more column of the keys, bf16: the rows that fill the last tile of 40 queries are zeros, and zero times -inf is
    no number (nor is it a term of these gradients; dq's column of the mask has none, by definition)"""
    low = torch.finfo(torch.bfloat16).min if low == "lowest" else -math.inf
    q, k, v, table, plan, dout, ref = _last_key_hidden(be, FEW, torch.bfloat16, low)
    a = [*be.to(q, k, v, table), _plan_on(be, plan)]
    out, lse = be.ops.rel_attention(*a, return_lse=True)
    _within(out, *ref["out"], "out")
    grads = dict(zip(("dq", "dk", "dv", "dtable"), be.ops.rel_attention_backward(*a, out, lse, be.to(dout))))
    for name, g in grads.items():
        cut = slice(1, None) if name == "dq" and low == -math.inf else slice(None)
        _within(g[..., cut], ref[name][0][..., cut], ref[name][1][..., cut], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", ["lowest", "-inf"])
@pytest.mark.parametrize("case", [FEW, MANY])
def test_rel_attention_key_hidden_by_a_column(be, case, low, dtype):
    """a mask as one more column of the keys: the lowest number of the type, or -inf (whose product with the zeros of dS leaves
    that column of dq without a value, by definition)"""
    low = torch.finfo(dtype).min if low == "lowest" else -math.inf
    q, k, v, table, plan, dout, ref = _last_key_hidden(be, case, dtype, low)
    a = [*be.to(q, k, v, table), _plan_on(be, plan)]
    out, lse = be.ops.rel_attention(*a, return_lse=True)
    _within(out, *ref["out"], "out")
    _within(lse, *ref["lse"], "lse")
    if case is MANY:
        return
    grads = dict(zip(("dq", "dk", "dv", "dtable"), be.ops.rel_attention_backward(*a, out, lse, be.to(dout))))
    for name, g in grads.items():
        cut = slice(1, None) if name == "dq" and low == -math.inf else slice(None)
        _within(g[..., cut], ref[name][0][..., cut], ref[name][1][..., cut], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [FEW, MANY])
def test_rel_attention_infinite_values(be, case, dtype):
    """an infinity in one column of v, two that meet in another, a NaN in a third: these columns, and nothing else, show it"""
    q, k, v, table, plan, lens, _ = _attn_inputs(case, dtype)
    ref = _attn_ref(q, k, v, table, plan, case[6], case[5] ** -0.5, *lens, None, dtype)
    v[:, 7, :, 3], v[:, 8, :, 4], v[:, 20, :, 4], v[:, 30, :, 5], v[:, 9, :, 6] = math.inf, math.inf, -math.inf, NAN, -math.inf
    out = be.ops.rel_attention(*be.to(q, k, v, table), _plan_on(be, plan), k_lens=be.to(lens[1])).cpu()
    assert bool((out[..., 3] == math.inf).all()) and bool((out[..., 6] == -math.inf).all())
    assert bool(out[..., 4].isnan().all()) and bool(out[..., 5].isnan().all())
    other = [c for c in range(case[5]) if c not in (3, 4, 5, 6)]
    _within(out[..., other], ref["out"][0][..., other], ref["out"][1][..., other], "out")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [FEW, MANY])
def test_rel_attention_nan_reaches_its_rows(be, case, dtype):
    """a NaN in a query shows in its row alone, one in a key in every row that sees it"""
    q, k, v, table, plan, lens, _ = _attn_inputs(case, dtype)
    ref = _attn_ref(q, k, v, table, plan, case[6], case[5] ** -0.5, *lens, None, dtype)
    kw = dict(k_lens=be.to(lens[1]))
    q[:, 5, 0, 1] = NAN
    out = be.ops.rel_attention(*be.to(q, k, v, table), _plan_on(be, plan), **kw).cpu()
    assert bool(out[:, 5, 0].isnan().all())
    rest = torch.ones(out.shape[:3], dtype=torch.bool)
    rest[:, 5, 0] = False
    _within(out[rest], ref["out"][0][rest], ref["out"][1][rest], "out")
    k[:, 11, :, 2] = NAN
    assert bool(be.ops.rel_attention(*be.to(q, k, v, table), _plan_on(be, plan), **kw).isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 35, 40, 1, 1, 96, True, 8, 20, False, [(35, 40, -5)]),
                                  (1, 3, 1030, 1, 1, 32, True, 8, 20, False, [(3, 1030, -1)]),      # keys in parts
                                  (1, 40, 40, 56, 28, 128, True, 8, 9, False, [(40, 40, -5)])])     # the kernel for many queries
def test_rel_attention_rows_without_keys_beside_an_infinity(be, case, dtype):
    """rows that stand before every key are zeros whatever the keys of their tile hold; so is a head whose buckets are all out"""
    q, k, v, table, plan, lens, _ = _attn_inputs(case, dtype)
    ref = _attn_ref(q, k, v, table, plan, True, case[5] ** -0.5, *lens, None, dtype)
    v[:, 0, :, 3] = math.inf
    a = be.to(q, k, v)
    kw = dict(causal=True, return_lse=True, q_start=be.to(lens[2]))
    out, lse = be.ops.rel_attention(*a, be.to(table), _plan_on(be, plan), **kw)
    first = -int(lens[2][0])
    assert bool((out[:, :first] == 0).all()) and bool((lse[..., :first] == -math.inf).all())
    assert bool((out[:, first:, :, 3] == math.inf).all())
    cols = [c for c in range(case[5]) if c != 3]
    _within(out[..., cols], ref["out"][0][..., cols], ref["out"][1][..., cols], "out")
    out, lse = be.ops.rel_attention(*a, be.to(torch.full_like(table, -math.inf)), _plan_on(be, plan), **kw)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 40, 40, 1, 1, 32, True, 8, 9, False, [(37, 40, -5)]),
                                  (1, 9, 300, 1, 1, 24, True, 8, 9, False, [(7, 300, -3)]),          # keys in parts
                                  (2, 40, 20, 2, 1, 64, False, 8, 9, True, [(33, 20, 0), (0, 20, 0)])])
def test_rel_attention_backward_rows_that_do_not_count_beside_an_infinity(be, case, dtype):
    """dq of rows behind the last query, and of rows that see no key, is zero whatever the keys and values hold"""
    q, k, v, table, plan, lens, dout = _attn_inputs(case, dtype)
    k[:, 0, :, 2], v[:, 0, :, 3], v[:, 1, :, 4] = math.inf, -math.inf, NAN
    a = [*be.to(q, k, v, table), _plan_on(be, plan)]
    kw = dict(causal=case[6], **dict(zip(("q_lens", "k_lens", "q_start"), be.to(*lens))))
    out, lse = be.ops.rel_attention(*a, return_lse=True, **kw)
    dq, dk, dv, dtable = be.ops.rel_attention_backward(*a, out, lse, be.to(dout), **kw)
    for b, (n, m, start) in enumerate(case[10]):
        unseen = max(0, -start) if case[6] else 0
        assert bool((out[b, n:] == 0).all()) and bool((out[b, :unseen] == 0).all())
        assert bool((dq[b, n:] == 0).all()) and bool((dq[b, :unseen] == 0).all())
        assert n == 0 or bool(dq[b, unseen:n].isnan().any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 40, 50, 2, 1, 32, True, 8, 9, False, [(40, 40, 0)]),
                                  (2, 20, 300, 2, 2, 24, True, 8, 9, False, [(20, 40, 20), (11, 6, -5)])])
def test_rel_attention_backward_keys_behind_the_last_query(be, case, dtype):
    """causal: what the rows behind the last query's position hold (a cache not filled yet) is not looked at"""
    q, k, v, table, plan, lens, dout = _attn_inputs(case, dtype)         # (NaN there)
    ref = _attn_ref(q, k, v, table, plan, True, case[5] ** -0.5, *lens, dout, dtype)
    a = [*be.to(q, k, v, table), _plan_on(be, plan)]
    kw = dict(causal=True, q_lens=be.to(lens[0]), q_start=be.to(lens[2]))
    out, lse = be.ops.rel_attention(*a, return_lse=True, **kw)
    _within(out, *ref["out"], "out")
    for name, g in zip(("dq", "dk", "dv", "dtable"), be.ops.rel_attention_backward(*a, out, lse, be.to(dout), **kw)):
        _within(g, *ref[name], name)


@pytest.mark.gpu
def test_rel_attention_sum_of_many_probabilities(hip):
    """the softmax sum over 32768 keys in one walk.  The values are 1 at 64 keys and 0 elsewhere, so that an output is a short sum
    over the long one.  T = 512 tiles are added onto a lane's running sum: rounding errors of u at its size then, independent, grow to
    u sqrt(T) / 3 = 7.5 u, over the two lanes of a row 5.3 u; a probability, the short sum, logarithms and the quotient add 3 u.
    (One probability after another: 16384 additions, 30 u.)  Bound: twice the former, 17 u."""
    L, H, D = 32768, 512, 24
    q, k = hip.to(_randn((1, 33, H, D), 51, 1.5)), hip.to(_randn((1, L, 8, D), 52))
    v = torch.zeros((1, L, 8, D), device=hip.device)
    v[:, -64:] = 1.0
    plan = _plan_on(hip, _attn_inputs(FEW, torch.float32)[4])
    table = torch.zeros((8, H), device=hip.device)
    out = hip.ops.rel_attention(q, k, v, table, plan)
    worst = []
    for h in range(0, H, 37):
        p = torch.softmax(q[0, :, h].double() @ k[0, :, h // 64].double().t() * D ** -0.5, -1)
        want = p[:, -64:].sum(-1, keepdim=True)
        worst.append(((out[0, :, h].double() - want) / want).square().mean())
    assert float(torch.stack(worst).mean().sqrt()) <= 17 * U


def test_second_derivatives_are_refused(be, monkeypatch):
    """the gradients come out of kernels that autograd cannot differentiate: asking for it raises, it does not drop the terms"""
    from occformer_amd import autograd as A
    monkeypatch.setattr(A, "get_ops", lambda: be.ops)
    q, k, v, table, plan, _, _ = _attn_inputs(FEW, torch.float32)
    q, k, v, table = (t.nan_to_num() for t in (q, k, v, table))
    w = torch.ones(32)
    x = [be.to(t.contiguous()).requires_grad_() for t in (q, k, v, table, w, w)]
    out = A.rel_attention(*x[:4], _plan_on(be, plan))
    g, = torch.autograd.grad(out.square().sum(), x[0], create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(g.sum() + x[0].sum(), x[0])
    for y in (g.square().sum(), g.sum() + x[0].sum()):
        with pytest.raises(RuntimeError, match="not differentiable again"):
            y.backward(retain_graph=True)
    qn, kn = A.qk_norm_rope(x[0], x[1], x[4], x[5])
    g, = torch.autograd.grad(qn.square().sum() + kn.sum(), x[0], create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(g.sum() + x[0].sum(), x[0])


def test_rel_attention_c_entry_refuses_a_workspace_off_16_bytes(be):
    """parts of the keys are written and read 16 bytes at a time"""
    import ctypes
    B, L, H, D = 1, 1030, 1, 32
    g = (ctypes.c_int64 * 17)(B, 1, L, H, H, D, 8, 9, *[D * H, D * H, D], *[L * D * H, D * H, D] * 2)
    lib, n = be.ops.lib, be.ops.lib.occf_rel_attn_workspace
    need = n(g, 0)
    assert need > 0
    q, k, v, table = be.to(_randn((B, 1, H, D), 1), _randn((B, L, H, D), 2), _randn((B, L, H, D), 3), _randn((8, H), 4))
    lut = _plan_on(be, _attn_inputs(FEW, torch.float32)[4]).lut
    out, ws = torch.empty_like(q), torch.empty((need + 4,), dtype=torch.float32, device=q.device)
    base = (-ws.data_ptr() % 16) // 4
    for off in (1, 2, 3):
        ptr = [q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), lut.data_ptr(), None, None, None, out.data_ptr(), None,
               ws[(base + off) % 4:].data_ptr()]
        assert (ptr[-1] % 16) != 0
        assert lib.occf_rel_attn_fwd(*ptr, need, g, 1.0, 0, 0, ctypes.c_void_p(0)) < 0


def test_rel_attention_backward_refuses_gradient_rows_too_far_apart(be):
    """rows of the gradient of the output lie Hq D elements apart, whatever the strides of q say (one head repeated)"""
    import ctypes
    for Hq, D, ok in ((1 << 19, 8, False), ((1 << 19) - 1, 8, True), (1 << 16, 64, False)):
        g = (ctypes.c_int64 * 17)(1, 2, 2, Hq, 1, D, 8, 9, *[2 * D, D, 0], *[2 * D, D, 0] * 2)
        for dtype in (0, 1):
            assert (be.ops.lib.occf_rel_attn_bwd_workspace(g, 0, dtype) > 0) == ok
            n = ctypes.c_void_p(16)
            if not ok:
                assert be.ops.lib.occf_rel_attn_bwd(*[n] * 16, 1 << 40, g, 1.0, 0, dtype, ctypes.c_void_p(0)) < 0
            assert be.ops.lib.occf_rel_attn_workspace(g, dtype) >= 0       # the forward has no such rows


def test_qk_norm_rope_weight_gradient_sums(be):
    """the weights' gradient over N = 10 000 rows, by its roundings (each u sqrt(1/3) 0.74 of its value in the mean square, for values
    spread over a binade).  Independent terms of size s leave s sqrt(k) behind k of them, so that a chain of n equal parts rounds as
    often as (n + 1) / 2 additions of the whole.  16 of a workgroup's 64 rows in a row: 8.5, two steps of pairs 2; 5 of 157
    workgroups 3, 8 of 32 such 4.5, pairs 2: together 20, and 0.5 u^2 of a term's own make a root of 0.5 + 20 * 0.18: 2.0 u s sqrt(N).
    (64 rows and 32 sums one after the other: 52 -> 3.1.)  Bound: half-way, over 6 seeds of two weights of 32 columns."""
    B, L, H, D = 1, 2500, 4, 32
    total = 0.0
    for seed in range(6):
        x, dz = _randn((2, B, L, H, D), 70 + seed, 2.0), _randn((2, B, L, H, D), 90 + seed)
        w = torch.ones(D)
        dw = be.ops.qk_norm_rope_backward(*be.to(x[0], x[1], w, w, dz[0], dz[1]))[2:]
        for i in (0, 1):
            xd = x[i].double()
            terms = dz[i].double() * xd * (xd.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            err = (dw[i].cpu().double() - terms.sum((0, 1, 2))) / (U * terms.square().sum((0, 1, 2)).sqrt())
            total += float(err.square().mean())
    assert (total / 12) ** 0.5 <= 2.6


@pytest.mark.parametrize("dtype,D", [(torch.float32, 6), (torch.bfloat16, 10), (torch.bfloat16, 24), (torch.float32, 128)])
def test_qk_norm_rope_takes_gradients_as_they_are(be, dtype, D):
    """contiguous gradients on 16 bytes go to the kernel whatever their rows' length, and their layout is checked once"""
    q, w = be.to(_randn((2, 5, 3, D), 1).to(dtype), torch.ones(D, dtype=dtype))
    dz = be.to(_randn((2, 5, 3, D), 2).to(dtype))
    args = (q, None, w, None, None, None, None, dz, None)
    plan, taken = be.ops._check_norm(*args, None, False, "qk_norm_rope_backward")
    assert taken[7] is dz
    before = be.ops.qk_norm_rope_backward(q, None, w, None, dz, None)
    assert be.ops._plan(be.ops._check_norm, args, None, False, "qk_norm_rope_backward")[0] is \
        be.ops._plan(be.ops._check_norm, args, None, False, "qk_norm_rope_backward")[0]
    off = torch.empty((dz.numel() + 1,), dtype=dtype, device=dz.device)[1:].view(dz.shape)
    off.copy_(dz)                                                        # off 16 bytes: copied, not refused
    for a, b in zip(before, be.ops.qk_norm_rope_backward(q, None, w, None, off, None)):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_relative_buckets_of_any_integer_type(dtype):
    """a radius that the distances' type cannot hold"""
    plan = RelativeBuckets(32, 400, True, device="cpu")
    top = min(torch.iinfo(dtype).max, 1000)
    d = torch.tensor([0, 1, 5, 100, top], dtype=dtype)
    assert torch.equal(plan.bucket(d), plan.bucket(d.long()))
    assert [int(plan.bucket(d)[i]) for i in range(5)] == [int(plan.lut[400 + min(int(x), 400)]) for x in d]
    if dtype != torch.uint8:
        assert torch.equal(plan.bucket(-d), plan.bucket(-d.long()))


def test_qk_norm_rope_c_entry_refuses_sizes_beyond_32_bits(be):
    """table rows and axis cuts are 32-bit numbers in the kernel"""
    import ctypes
    q, w = be.to(_randn((1, 4, 2, 8), 1), torch.ones(8))
    cos, sin = be.to(torch.ones(8, 4), torch.zeros(8, 4))
    pos, out = be.to(torch.zeros((4, 2), dtype=torch.int32)), torch.empty_like(q)
    for rows, cuts in ((1 << 31, (2, 4)), ((1 << 32) + 8, (2, 4)), (8, (2, (1 << 32) + 2)), (8, ((1 << 32) + 1, (1 << 32) + 4))):
        g = (ctypes.c_int64 * 17)(1, 4, 2, 0, 8, 8, rows, 2, *cuts, 0, 64, 16, 8, 0, 0, 0)
        ptr = [t if t is None else t.data_ptr() for t in (q, None, w, None, cos, sin, pos, out, None)]
        assert be.ops.lib.occf_qk_norm_rope_fwd(*ptr, g, 1e-6, 0, 0, ctypes.c_void_p(0)) < 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 9, 640, 2, 1, 32, True, 128, 512, False, [(9, 640, 631)]),
                                  (1, 40, 70, 2, 2, 128, False, 128, 512, True, [(40, 70, -300)]),
                                  (1, 33, 40, 1, 1, 64, False, 128, 100, True, None)])
def test_rel_attention_most_buckets_and_widest_radius(be, case, dtype):
    _check_attention(be, case, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rel_attention_more_sequences_than_parts_are_counted_for(be, dtype):
    n = [(7 * b) % 34 for b in range(520)]
    _check_attention(be, (520, 1, 33, 2, 1, 8, True, 8, 40, False, [(1, m, m - 1) for m in n]), dtype, backward=False)


@pytest.mark.parametrize("case", [(1, 40, 200, 2, 2, 32, False, 32, 40, True, None), (4, 1, 1700, 8, 2, 64, True, 8, 40, False, None),
                                  (3, 5, 300, 8, 2, 128, True, 8, 40, False, [(5, 300, 295), (5, 129, 124), (5, 200, 195)])])
def test_rel_attention_few_queries_round_once(be, case):
    """bf16, few queries: no further off, in the mean square, than the last rounding of the exact value and a tenth (what else there
    is, 2^-16 of a probability and sums in 32 bits, would have to be 0.45 of it to show)"""
    q, k, v, table, plan, lens, _ = _attn_inputs(case, torch.bfloat16)
    if case[10] is None:
        lens[2] += case[2] - case[1]
    want = _attn_ref(q, k, v, table, plan, case[6], case[5] ** -0.5, *lens, None, torch.bfloat16)["out"][0]
    out = be.ops.rel_attention(*be.to(q, k, v, table), _plan_on(be, plan), causal=case[6], k_lens=be.to(lens[1]), q_start=be.to(lens[2]))
    assert float((out.cpu().double() - want).norm()) <= 1.1 * float((want.bfloat16().double() - want).norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter", [False, True])
def test_qk_norm_rope_infinity_stays_in_its_column(be, inter, dtype):
    """a row with an infinity: its root mean square is infinite, so every finite column comes out as zero and the infinite one as NaN,
    which the rotation takes to its partner, but the columns that are not turned have none"""
    D, half = 32, 4
    q, w = _randn((1, 3, 1, D), 1).to(dtype), torch.ones(D, dtype=dtype)
    q[0, 1, 0, 20] = math.inf
    for rot in (None, half):
        cos, sin = (None, None) if rot is None else be.to(torch.full((4, half), 0.6), torch.full((4, half), 0.8))
        out = be.ops.qk_norm_rope(be.to(q), None, be.to(w), None, cos, sin, interleaved=inter)[0].cpu()
        assert bool(out[0, 1, 0, 20].isnan()) and int((out[0, 1, 0] == 0).sum()) == D - 1
        assert bool(out[0, 0].isfinite().all()) and bool(out[0, 2].isfinite().all())


def test_gradients_kept_for_a_graph_can_be_changed_in_place(be, monkeypatch):
    """gradients asked for with create_graph are tensors of their own: scaling one in place is nobody's business"""
    from occformer_amd import autograd as A
    monkeypatch.setattr(A, "get_ops", lambda: be.ops)
    q, k, v, table, plan, _, _ = _attn_inputs(FEW, torch.float32)
    x = [be.to(t.nan_to_num().contiguous()).requires_grad_() for t in (q, k, v, table)]
    plain = torch.autograd.grad(A.rel_attention(*x, _plan_on(be, plan)).square().sum(), x)
    kept = torch.autograd.grad(A.rel_attention(*x, _plan_on(be, plan)).square().sum(), x, create_graph=True)
    for a, b in zip(plain, kept):
        assert torch.equal(a, b)
        b.mul_(2.0)
        assert torch.equal(2.0 * a, b)
