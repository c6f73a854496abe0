"""What the position operators of the attention path are timed on: per-head norms of queries and keys with the position
rotation (``qk_norm_rope``) and attention with a learned relative position bias by buckets (``rel_attention``), each with
its backward pass, the attention also for single queries over a long set of keys.

``run`` computes them in elementary torch operations in 32 bits, or (``own``) through ``occformer_amd``'s entry points;
``exact`` restates the definitions in 64 bits."""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
EPS = 1e-6


def listed():
    return [
        # one object query added to the decoder's set: 8 heads of 24, the smallest call there is
        dict(name="norm token f32", op="norm", B=1, L=1, Hq=8, Hk=8, D=24, axes=1, dtype=F32),
        # a long prompt's queries and shared keys, bfloat16
        dict(name="norm prompt bf16", op="norm", B=2, L=8192, Hq=32, Hk=8, D=128, axes=1, dtype=BF16),
        # training on a 100 x 100 grid of tokens of the encoder (128 channels, 4 heads) with (x, y, z) positions
        dict(name="norm train voxels f32", op="norm_train", B=1, L=10000, Hq=4, Hk=4, D=32, axes=3, dtype=F32),
        # training on packed sequences, shared keys
        dict(name="norm train bf16", op="norm_train", B=4, L=4095, Hq=16, Hk=4, D=64, axes=1, dtype=BF16),
        # the occupancy decoder's 100 queries among themselves
        dict(name="attn queries f32", op="attn", B=1, Lq=100, Lk=100, Hq=8, Hk=8, D=24, causal=False, ragged=False,
             buckets=32, radius=128, dtype=F32),
        # a batch of 50 x 50 bird's-eye-view token maps, the last ones cropped
        dict(name="attn bev f32", op="attn", B=4, Lq=2500, Lk=2500, Hq=4, Hk=4, D=32, causal=False, ragged=True,
             buckets=32, radius=128, dtype=F32),
        # a long prompt, causal, shared keys
        dict(name="attn prompt bf16", op="attn", B=1, Lq=8192, Lk=8192, Hq=16, Hk=2, D=128, causal=True, ragged=False,
             buckets=32, radius=128, dtype=BF16),
        # training at the width of the pixel decoder (192 channels, 8 heads)
        dict(name="attn train f32", op="attn_train", B=2, Lq=1000, Lk=1000, Hq=8, Hk=8, D=24, causal=False, ragged=False,
             buckets=32, radius=128, dtype=F32),
        # training on padded sequences of odd length
        dict(name="attn train ragged bf16", op="attn_train", B=3, Lq=777, Lk=777, Hq=12, Hk=12, D=64, causal=False,
             ragged=True, buckets=32, radius=128, dtype=BF16),
        # training on long sequences, causal, shared keys: the most work
        dict(name="attn train causal bf16", op="attn_train", B=2, Lq=4096, Lk=4096, Hq=16, Hk=4, D=64, causal=True,
             ragged=False, buckets=32, radius=128, dtype=BF16),
        # one new query against a few hundred kept keys
        dict(name="decode short f32", op="attn", B=1, Lq=1, Lk=333, Hq=8, Hk=8, D=24, causal=True, ragged=False,
             buckets=32, radius=128, dtype=F32),
        # one new token of each of 16 sequences against kept keys of differing length
        dict(name="decode batch bf16", op="attn", B=16, Lq=1, Lk=8192, Hq=32, Hk=8, D=128, causal=True, ragged=True,
             buckets=32, radius=128, dtype=BF16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_train", "attn", "attn_train", "decode"])
    dtype = rng.choice([F32, BF16])
    D = rng.choice([24, 32, 64, 96, 128])
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hq = Hk * rng.choice([1, 1, 2, 4])
    if op in ("norm", "norm_train"):
        B = rng.randint(1, 4)
        L = _log_int(rng, 1, max(1, min(16384, (1 << 26) // (B * (Hq + Hk) * D))))
        return dict(op=op, B=B, L=L, Hq=Hq, Hk=Hk, D=D, axes=rng.choice([1, 3]), dtype=dtype)
    common = dict(Hq=Hq, Hk=Hk, D=D, ragged=rng.random() < 0.5, buckets=rng.choice([8, 32, 64]),
                  radius=rng.choice([40, 128, 500]), dtype=dtype)
    if op == "decode":
        B = rng.randint(1, 16)
        Lk = _log_int(rng, 1, min(32768, (1 << 27) // (B * Hk * D)))
        return dict(op="attn", B=B, Lq=min(Lk, rng.choice([1, 1, 1, 2, 5])), Lk=Lk, causal=True, **common)
    B = rng.randint(1, 3)
    most = 2 * 16 * 4096 * 4096 * 64 // (4 if dtype == F32 else 2)
    L = _log_int(rng, 2, min(4096, int(math.sqrt(most / (B * Hq * D)))))
    Lq = L if rng.random() < 0.7 else max(1, L // rng.randint(2, 9))
    return dict(op=op, B=B, Lq=Lq, Lk=L, causal=rng.random() < 0.5, **common)


# ------------------------------------------------------------------------------------------------------- inputs
def _axis_dims(case):
    """pairs of columns that each position axis turns"""
    half, a = case["D"] // 2, case["axes"]
    return tuple(half // a + (1 if i < half % a else 0) for i in range(a))


def _rows(case):
    """(queries, keys, position of the first query) of every sequence; where there are fewer queries than keys the last
    query stands at the last key. A ragged batch of three or more has an empty place at its end."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    lens = [Lk - (b * Lk) // B if case["ragged"] else Lk for b in range(B)]
    if case["ragged"] and B > 2:
        lens[-1] = 0
    if Lq == Lk:
        return [(n, n, 0) for n in lens]
    return [(min(Lq, n), n, n - min(Lq, n)) for n in lens]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == BF16 else torch.float32


def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, device="cuda", generator=gen) * scale


def _norm_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, L, Hq, Hk, D, axes = (case[k] for k in ("B", "L", "Hq", "Hk", "D", "axes"))
    dt = _dtype(case)
    # queries, keys and values come out of one projection: the operator reads column blocks of its rows
    qkv = _normal((B, L, (Hq + 2 * Hk) * D), gen, 2.0).to(dt)
    s = dict(q=qkv[..., :Hq * D].unflatten(-1, (Hq, D)), k=qkv[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D)),
             qw=(1 + _normal((D,), gen, 0.1)).to(dt), kw=(1 + _normal((D,), gen, 0.1)).to(dt))
    if axes == 1:
        first = torch.randint(0, 16384, (B, 1), device="cuda", generator=gen)
        s["positions"] = (first + torch.arange(L, device="cuda")).int()
        s["length"] = 32768
    else:
        s["positions"] = torch.stack([torch.randint(0, n, (B, L), device="cuda", generator=gen) for n in (200, 200, 16)],
                                     -1).int()
        s["length"] = 200
    if case["op"] == "norm_train":
        s["dq"] = _normal((B, L, Hq, D), gen).to(dt)
        s["dk"] = _normal((B, L, Hk, D), gen).to(dt)
    return s


def _angles(case, length):
    """angles in 64 bits, [length, D / 2]: position * base^(-column / columns of the axis)"""
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in _axis_dims(case)])
    return (torch.arange(length, dtype=torch.float64)[:, None] * freq).cuda()


def _edges(n, radius):
    """first distances of the logarithmic buckets e + 1 .. n - 1 (e = n // 2 exact ones): the least integer d with
    (d / e)^(n - e) >= (radius / e)^m, in whole numbers"""
    e = n // 2
    got, d = [], e
    for m in range(1, n - e):
        while d ** (n - e) < e ** (n - e - m) * radius ** m:
            d += 1
        got.append(d)
    return e, got


def _attn_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    dt = _dtype(case)
    kv = _normal((B, Lk, 2 * Hk * D), gen).to(dt)
    s = dict(q=_normal((B, Lq, Hq, D), gen, 1.5).to(dt), k=kv[..., :Hk * D].unflatten(-1, (Hk, D)),
             v=kv[..., Hk * D:].unflatten(-1, (Hk, D)), table=_normal((case["buckets"], Hq), gen, 0.7).to(dt))
    rows = torch.tensor(_rows(case), dtype=torch.int32, device="cuda")
    s["q_lens"], s["k_lens"], s["q_start"] = (rows[:, i].contiguous() for i in range(3))
    if case["op"] == "attn_train":
        s["dout"] = _normal((B, Lq, Hq, D), gen).to(dt)
    return s


def prepare(case, seed):
    s = _norm_inputs(case, seed) if case["op"].startswith("norm") else _attn_inputs(case, seed)
    s["case"] = case
    if case["op"].startswith("norm"):
        a = _angles(case, s.pop("length"))
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()         # the tables that a program keeps
    elif own:
        from occformer_amd.position import RelativeBuckets
        s["plan"] = RelativeBuckets(case["buckets"], case["radius"], bidirectional=not case["causal"], device="cuda")
    else:
        n = case["buckets"] if case["causal"] else case["buckets"] // 2
        e, edges = _edges(n, case["radius"])
        s["exact_buckets"], s["edges"] = e, torch.tensor(edges, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------- the plain form
def _axis_of(case, device):
    return torch.repeat_interleave(torch.arange(case["axes"], device=device),
                                   torch.tensor(_axis_dims(case), device=device), output_size=case["D"] // 2)


def _turns(s, case):
    """cos and sin of every token's columns, [B, L, 1, D / 2]"""
    pos = s["positions"].long()
    if case["axes"] == 1:
        return s["cos"][pos].unsqueeze(2), s["sin"][pos].unsqueeze(2)
    rows = pos[..., _axis_of(case, pos.device)]
    cols = torch.arange(case["D"] // 2, device=pos.device)
    return s["cos"][rows, cols].unsqueeze(2), s["sin"][rows, cols].unsqueeze(2)


def _norm_plain(x, w, cos, sin):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _norm_plain_backward(x, w, dz, cos, sin):
    x, w, dz = x.float(), w.float(), dz.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n = x * r
    a, b = dz.chunk(2, -1)
    dy = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
    g = dy * w
    return r * (g - n * (g * n).mean(-1, keepdim=True)), (dy * n).sum((0, 1, 2))


def _run_norm_plain(s, case):
    dt = _dtype(case)
    cos, sin = _turns(s, case)
    got = dict(q=_norm_plain(s["q"], s["qw"], cos, sin).to(dt), k=_norm_plain(s["k"], s["kw"], cos, sin).to(dt))
    if case["op"] == "norm_train":
        dq, dqw = _norm_plain_backward(s["q"], s["qw"], s["dq"], cos, sin)
        dk, dkw = _norm_plain_backward(s["k"], s["kw"], s["dk"], cos, sin)
        got.update(dq=dq.to(dt), dk=dk.to(dt), dqw=dqw.to(dt), dkw=dkw.to(dt))
    return got


def _bucket_index(s, case):
    """bucket of every (query, key) pair and whether the pair counts, [B, Lq, Lk]"""
    dev = s["q"].device
    i = torch.arange(case["Lq"], device=dev)
    j = torch.arange(case["Lk"], device=dev)
    rel = j[None, None, :] - (s["q_start"].long()[:, None] + i)[:, :, None]
    keep = (j[None, None, :] < s["k_lens"][:, None, None]) & (i[None, :, None] < s["q_lens"][:, None, None])
    if case["causal"]:
        keep = keep & (rel <= 0)
        dist = (-rel).clamp(min=0)
    else:
        dist = rel.abs()
    e = s["exact_buckets"]
    bucket = torch.where(dist < e, dist, e + torch.bucketize(dist, s["edges"], right=True))
    if not case["causal"]:
        bucket = bucket + torch.where(rel > 0, case["buckets"] // 2, 0)
    return bucket, keep


def _run_attn_plain(s, case):
    dt = _dtype(case)
    B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    G, scale = Hq // Hk, D ** -0.5
    bucket, keep = _bucket_index(s, case)
    q = s["q"].float().permute(0, 2, 1, 3)
    k = s["k"].float().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    v = s["v"].float().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    bias = s["table"].float()[bucket].permute(0, 3, 1, 2)
    t = (q @ k.transpose(-1, -2)) * scale + bias
    t = t.masked_fill(~keep[:, None], float("-inf"))
    m = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(m == float("-inf"), 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    got = dict(out=out.permute(0, 2, 1, 3).to(dt))
    if case["op"] == "attn_train":
        do = s["dout"].float().permute(0, 2, 1, 3)
        dv = p.transpose(-1, -2) @ do
        dp = do @ v.transpose(-1, -2)
        ds = p * (dp - (do * out).sum(-1, keepdim=True))
        dq = ds @ k * scale
        dk = ds.transpose(-1, -2) @ q * scale
        # one product a query row with the rows' buckets as 0 / 1 columns, then the sum over rows
        hot = (bucket[..., None] == torch.arange(case["buckets"], device=q.device)).float()
        dtable = torch.bmm(ds.permute(0, 2, 1, 3).reshape(B * Lq, Hq, Lk), hot.reshape(B * Lq, Lk, -1)).sum(0).t()
        got.update(dq=dq.permute(0, 2, 1, 3).to(dt), dk=dk.unflatten(1, (Hk, G)).sum(2).permute(0, 2, 1, 3).to(dt),
                   dv=dv.unflatten(1, (Hk, G)).sum(2).permute(0, 2, 1, 3).to(dt), dtable=dtable.to(dt))
    return got


# ------------------------------------------------------------------------------------------------------- the operators
def _run_norm_own(s, case):
    from occformer_amd.ops import get_ops
    ops = get_ops()
    rot = dict(cos=s["cos"], sin=s["sin"], positions=s["positions"], eps=EPS,
               axis_dims=None if case["axes"] == 1 else _axis_dims(case))
    q, k = ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], **rot)
    got = dict(q=q, k=k)
    if case["op"] == "norm_train":
        dq, dk, dqw, dkw = ops.qk_norm_rope_backward(s["q"], s["k"], s["qw"], s["kw"], s["dq"], s["dk"], **rot)
        got.update(dq=dq, dk=dk, dqw=dqw, dkw=dkw)
    return got


def _run_attn_own(s, case):
    from occformer_amd.ops import get_ops
    ops = get_ops()
    rows = dict(causal=case["causal"], q_lens=s["q_lens"], k_lens=s["k_lens"], q_start=s["q_start"])
    if case["op"] == "attn":
        return dict(out=ops.rel_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], **rows))
    out, lse = ops.rel_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], return_lse=True, **rows)
    dq, dk, dv, dtable = ops.rel_attention_backward(s["q"], s["k"], s["v"], s["table"], s["plan"], out, lse, s["dout"],
                                                    **rows)
    return dict(out=out, dq=dq, dk=dk, dv=dv, dtable=dtable)


def run(state):
    case = state["case"]
    if case["op"].startswith("norm"):
        return _run_norm_own(state, case) if own else _run_norm_plain(state, case)
    return _run_attn_own(state, case) if own else _run_attn_plain(state, case)


# ------------------------------------------------------------------------------------------------------- work, 64 bits
def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"].startswith("norm"):
        rows = case["B"] * case["L"] * (case["Hq"] + case["Hk"])
        table = case["B"] * case["L"] * case["D"] * 4
        if case["op"] == "norm":
            return {"bytes": 2 * rows * case["D"] * size + table, "flops": 8 * rows * case["D"]}
        return {"bytes": 5 * rows * case["D"] * size + table, "flops": 24 * rows * case["D"]}
    pairs = 0
    for n, m, start in _rows(case):
        pairs += sum(min(m, start + i + 1) for i in range(n)) if case["causal"] else n * m
    q = case["B"] * case["Lq"] * case["Hq"] * case["D"] * size
    kv = sum(m for _, m, _ in _rows(case)) * case["Hk"] * case["D"] * size
    if case["op"] == "attn":
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * case["Hq"] * case["D"]}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * case["Hq"] * case["D"]}


def _norm_exact(case, seed):
    s = _norm_inputs(case, seed)
    angle = _angles(case, s["length"])
    pos = s["positions"].long().reshape(case["B"], case["L"], case["axes"])
    parts, at = [], 0
    for a, n in enumerate(_axis_dims(case)):
        parts.append(angle[pos[..., a]][..., at:at + n])
        at += n
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.cat(parts, -1)).unsqueeze(2)
    half, got = case["D"] // 2, {}
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "w"].double()
        inv = (x.square().sum(-1, keepdim=True) / case["D"] + EPS) ** -0.5
        y = x * inv * w
        z = torch.complex(y[..., :half], y[..., half:]) * turn
        got[name] = torch.cat([z.real, z.imag], -1)
        if case["op"] == "norm_train":
            d = s["d" + name].double()
            back = torch.complex(d[..., :half], d[..., half:]) * turn.conj()
            dy = torch.cat([back.real, back.imag], -1)
            got["d" + name + "w"] = (dy * x * inv).flatten(0, 2).sum(0)
            dn = dy * w
            got["d" + name] = dn * inv - x * inv ** 3 * ((dn * x).sum(-1, keepdim=True) / case["D"])
    return got


def _buckets_exact(case, rel):
    """bucket of every distance in ``rel`` (a list of ints), by its definition"""
    n = case["buckets"] if case["causal"] else case["buckets"] // 2
    e, R, got = n // 2, case["radius"], []
    for r in rel:
        d = max(0, -r) if case["causal"] else abs(r)
        b = d
        if d >= e:
            b = e + max(m for m in range(n - e) if min(d, R) ** (n - e) >= e ** (n - e - m) * R ** m)
        got.append(b + (n if r > 0 and not case["causal"] else 0))
    return got


def _attn_exact(case, seed):
    s = _attn_inputs(case, seed)
    Lq, Lk, Hq, D, R = case["Lq"], case["Lk"], case["Hq"], case["D"], case["radius"]
    G, scale = Hq // case["Hk"], 1 / math.sqrt(D)
    of = torch.tensor(_buckets_exact(case, range(-R, R + 1)), device="cuda")
    got = dict(out=torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"))
    train = case["op"] == "attn_train"
    if train:
        for name in ("q", "k", "v", "table"):
            got["d" + name] = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
    for b, (n, m, start) in enumerate(_rows(case)):
        if not n or not m:
            continue
        rel = torch.arange(m, device="cuda")[None] - torch.arange(start, start + n, device="cuda")[:, None]
        bucket = of[rel.clamp(-R, R) + R]
        for h in range(Hq):
            q, k, v = s["q"][b, :n, h].double(), s["k"][b, :m, h // G].double(), s["v"][b, :m, h // G].double()
            t = q @ k.t() * scale + s["table"][:, h].double()[bucket]
            if case["causal"]:
                t = t.masked_fill(rel > 0, -math.inf)
            p = torch.softmax(t, -1)
            got["out"][b, :n, h] = p @ v
            if train:
                do = s["dout"][b, :n, h].double()
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                got["dq"][b, :n, h] = ds @ k * scale
                got["dk"][b, :m, h // G] += ds.t() @ q * scale
                got["dv"][b, :m, h // G] += p.t() @ do
                got["dtable"][:, h] += torch.bincount(bucket.flatten(), ds.flatten(), case["buckets"])
    return got


def exact(case, seed):
    return _norm_exact(case, seed) if case["op"].startswith("norm") else _attn_exact(case, seed)
