"""Host-side tables of the position operators (``ops.qk_norm_rope``, ``ops.rel_attention``): made once, kept by the program.

``rotary_table``     cosines and sines of every position's angles (64-bit angles, rounded once)
``RelativeBuckets``  the bucket of every relative distance, as a table over the clamped distances
"""
import torch


def rotary_table(length, rot_dim, base=10000.0, axis_dims=None, device="cuda"):
    """cos, sin fp32 [length, rot_dim / 2] for positions 0 .. length - 1.  Column c of an axis with n columns turns by
    position * base^(-c / n); ``axis_dims`` splits the rot_dim / 2 columns over up to three axes (x, y, z of a voxel), in
    order, every axis with frequencies of its own.  The angles are formed in 64 bits: at position 10^6 a 32-bit angle is
    off by up to 0.03."""
    half = rot_dim // 2
    dims = (half,) if axis_dims is None else tuple(int(n) for n in axis_dims)
    if rot_dim % 2 or half < 1 or length < 1:
        raise ValueError(f"rotary_table: rot_dim {rot_dim} must be even and positive, length {length} positive")
    if sum(dims) != half or not 1 <= len(dims) <= 3 or min(dims) < 1:
        raise ValueError(f"rotary_table: axis_dims {dims} must be one to three column counts that sum to {half}")
    freq = torch.cat([float(base) ** (-torch.arange(n, dtype=torch.float64) / n) for n in dims])
    angle = torch.arange(length, dtype=torch.float64)[:, None] * freq
    return angle.cos().float().to(device), angle.sin().float().to(device)


class RelativeBuckets:
    """Logarithmic buckets of the distance key - query.  ``bidirectional``: half of the buckets for keys at or before the
    query, half for keys behind it (offset ``num_buckets / 2``); else all for keys at or before it (keys behind it share
    bucket 0).  Of a direction's n buckets the first e = n // 2 hold one distance each; bucket e + m starts at the least
    integer d with (d / e)^(n - e) >= (max_distance / e)^m, and the last one takes every distance from its edge on.  The edges
    come from whole-number arithmetic: a 32-bit logarithm puts distances next to an edge into the bucket beside it.

    ``radius`` = ``max_distance``: every distance at or beyond it is in the outermost bucket of its side.
    ``lut`` int32 [2 radius + 1] on the device: bucket of the distance index - radius."""

    def __init__(self, num_buckets=32, max_distance=128, bidirectional=True, device="cuda"):
        n = num_buckets // 2 if bidirectional else num_buckets
        if num_buckets > 128 or n < 2 or (bidirectional and num_buckets % 2):
            raise ValueError(f"RelativeBuckets: num_buckets {num_buckets} must be at most 128 and leave two or more a side")
        exact = n // 2
        if not exact < max_distance <= 512:
            raise ValueError(f"RelativeBuckets: max_distance {max_distance} must lie in ({exact}, 512]")
        self.num_buckets, self.radius, self.bidirectional = int(num_buckets), int(max_distance), bool(bidirectional)
        edges, d = [], exact
        for m in range(1, n - exact):
            while d ** (n - exact) < exact ** (n - exact - m) * self.radius ** m:
                d += 1
            edges.append(d)
        self.edges = tuple(edges)
        side = [d if d < exact else exact + sum(d >= t for t in edges) for d in range(self.radius + 1)]
        after = [n + b for b in side[1:]] if bidirectional else [0] * self.radius
        self.lut = torch.tensor(side[::-1] + after, dtype=torch.int32, device=device)

    def bucket(self, distance):
        """bucket of every entry of an integer tensor of distances (key - query)"""
        return self.lut[distance.long().clamp(-self.radius, self.radius) + self.radius]
