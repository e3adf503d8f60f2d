"""What goes with the attention layers: buckets of relative positions, rotation angles, and clipping
of a network's gradients.  No counterpart in the reference."""
import math

import torch

from .. import _C


def distance_buckets(num_buckets, reach=None, circle=None, device=None):
    """Buckets of the relative positions key - query: half of them for each sign; half of those for
    the near distances, one each, and the rest for the farther ones by their logarithm.

    `reach`: positions on a line; distances from there on share the last bucket.
    `circle`: positions on a circle of so many places, as the columns of an equirectangular image;
    the distance is the shorter way round, its sign the way's.
    -> (buckets int32, zero): the entry of difference d is zero + d, the ends standing for all
    beyond."""
    assert (reach is None) != (circle is None), 'Give either reach or circle'
    assert num_buckets >= 4 and num_buckets % 4 == 0, 'Number of buckets must be a multiple of 4'
    span = reach if circle is None else circle - 1
    assert span >= 1, 'Positions must differ'
    difference = torch.arange(-span, span + 1, dtype=torch.float64)
    away = difference.abs()
    if circle is None:
        ahead = difference > 0
        last = reach
    else:
        round_the_other_way = circle - away
        # (half a circle away counts as behind, as 0 does)
        ahead = difference % circle * 2 < circle
        ahead &= difference != 0
        away = torch.minimum(away, round_the_other_way)
        last = circle // 2
    half, near = num_buckets // 2, num_buckets // 4
    far = torch.log(away.clamp_min(near) / near) / math.log(max(last, near + 1) / near)
    far = (near + far * (half - near)).floor().clamp_max(half - 1)
    bucket = torch.where(away < near, away, far) + half * ahead
    return bucket.to(torch.int32).to(device), span


def rotation_table(places, rotated, base=10000.0, circle=False, device=None):
    """cos and sin (float32, [places, rotated / 2]) of the angles that QKNormRotation turns the pairs
    of a place by: place * base ** -(2 f / rotated); or, with `circle`, whole turns over all places,
    f + 1 of them for pair f, so that the last place is next to the first."""
    assert rotated % 2 == 0, 'Values are turned in pairs'
    place = torch.arange(places, dtype=torch.float64)[:, None]
    pair = torch.arange(rotated // 2, dtype=torch.float64)[None]
    if circle:
        angle = 2 * math.pi * (place * (pair + 1) % places) / places
    else:
        angle = place * base ** (-2 * pair / max(rotated, 1))
    return angle.cos().float().to(device), angle.sin().float().to(device)


def clip_grad_norm_(parameters, max_norm, eps=1e-6):
    """Scales the gradients of the parameters in place so that the norm of all of them together is at
    most max_norm; -> that norm before (float32 scalar where the parameters are; 0 where there is no
    gradient).
    Gradients are float32 or bfloat16, on one GPU; one that is not contiguous is copied and back."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    # (a gradient that several have, or a parameter that is given twice, counts once)
    grads = list(dict.fromkeys(p.grad for p in parameters if p.grad is not None))
    if not grads:
        return torch.zeros((), dtype=torch.float32,
                           device=parameters[0].device if parameters else None)
    with torch.no_grad():
        dense = [g if g.is_contiguous() else g.contiguous() for g in grads]
        norm = _C.clip_grad_norm(dense, max_norm, eps)
        for g, d in zip(grads, dense):
            if d is not g:
                g.copy_(d)
    return norm
