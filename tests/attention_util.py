"""Plain 64-bit implementations of the attention operators and the error
bounds of the kernels' arithmetic, for their tests."""
import torch


def half_step(dtype):
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Largest absolute error of rounding a value below the normal range."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v in 64 bits for one head, and a bound of the
    kernel's error.

    q [nq, d], k and v [nk, d], seen [nq, nk] bool. A row that sees nothing is
    zeros. With u = half_step, the kernel's errors are
      * each probability rounded to the element type: u p (below the normal
        range an absolute step, against row sums of at least 1): at most
        u sum(p |v|) / l + tiny sum(|v|);
      * each score summed in f32 over d products and scaled: at most
        e = scale (d + 2) 2^-24 sum(|q| |k|), plus 2^-21 for the exponential
        and its argument's rounding (2^-24 |c s| there: |c s| 2^-23), which
        moves p and its share of l by that factor each;
      * the f32 sums over nk keys: nk 2^-24 relative, twice;
      * the result's own rounding: u |y|, or tiny.
    """
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    z = (q @ k.T) * scale
    z = torch.where(seen, z, -torch.inf)
    top = z.amax(-1, keepdim=True) if z.shape[1] else z.new_zeros(z.shape[0], 1)
    p = torch.where(seen, torch.exp(z - torch.where(top.isinf(), 0.0, top)), 0.0)
    l = p.sum(-1, keepdim=True)
    some = seen.any(-1, keepdim=True)
    l = torch.where(some, l, 1.0)
    visible = seen.any(0)[:, None]
    vz = torch.where(visible, v, 0.0)
    y = p @ vz / l
    weight = p @ vz.abs() / l
    mag = torch.where(seen, (q.abs() @ k.abs().T) * scale, 0.0)
    mag = mag.amax(-1, keepdim=True) if z.shape[1] else mag.new_zeros(mag.shape[0], 1)
    n, d = z.shape[1], q.shape[1]
    u = half_step(dt)
    e = 2 * ((d + 2) * 2.0 ** -24 * mag + 2.0 ** -21 + 2 * 1.45 * mag * 2.0 ** -23) + 4 * (n + 8) * 2.0 ** -24
    far = tiny(dt) * (1 + seen.double() @ vz.abs()) * 2.0 ** 1
    return y, (u + e) * weight + u * y.abs() + u * u * weight + far + e * weight


def causal_seen(nq, nk, device, causal=True):
    if not causal:
        return torch.ones(nq, nk, dtype=torch.bool, device=device)
    i = torch.arange(nq, device=device)[:, None]
    return torch.arange(nk, device=device)[None] <= i + nk - nq


def packed(q, k, v, nq, nk, scale, causal=True):
    """The rows of all sequences, one after another, and their error bound."""
    heads, kv = q.shape[1], k.shape[1]
    y = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    a = b = 0
    for m, n in zip(nq, nk):
        seen = causal_seen(m, n, q.device, causal)
        for h in range(heads):
            c = h // (heads // kv)
            y[a:a + m, h], bound[a:a + m, h] = attend(q[a:a + m, h], k[b:b + n, c], v[b:b + n, c], seen,
                                                      scale)
        a, b = a + m, b + n
    return y, bound


def prefix(q, pk, pv, kp, vp, lens, scale, pages=None):
    batch, steps, heads, d = q.shape
    kv, size = pk.shape[1], kp.shape[1]
    y = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    for b in range(batch):
        n = int(lens[b])
        j = torch.arange(n, device=q.device)
        at = torch.full_like(j, b) if pages is None else pages[b].long()[j // size]
        k = torch.cat([pk, kp[at, j % size]])
        v = torch.cat([pv, vp[at, j % size]])
        seen = causal_seen(steps, n, q.device)
        seen = torch.cat([torch.ones(steps, pk.shape[0], dtype=torch.bool, device=q.device), seen], 1)
        for h in range(heads):
            c = h // (heads // kv)
            y[b, :, h], bound[b, :, h] = attend(q[b, :, h], k[:, c], v[:, c], seen, scale)
    return y, bound


def norm_rope(x, weight, eps, table, positions, sections, interleaved):
    """Head norm and rotation in 64 bits, and a bound of the f32 arithmetic:
    the mean's sum of d squares and the inverse root, (d + 8) 2^-24 relative,
    three products and one sum, 4 2^-24 of the terms' magnitudes; then one
    rounding to the element type."""
    dt, d = x.dtype, x.shape[-1]
    rot = table.shape[1]
    half = rot // 2
    z = x.double()
    if weight is not None:
        z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps) * weight.double()
    pos = positions.long().reshape(-1, x.shape[0])
    y, mag = z.clone(), z.abs()
    i = 0
    for axis, count in enumerate(sections or [half]):
        for i in range(i, i + count):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            t = table.double()[pos[axis]]
            c, s = t[:, None, i], t[:, None, half + i]
            y[..., a] = z[..., a] * c - z[..., b] * s
            y[..., b] = z[..., b] * c + z[..., a] * s
            mag[..., a] = (z[..., a] * c).abs() + (z[..., b] * s).abs()
            mag[..., b] = (z[..., b] * c).abs() + (z[..., a] * s).abs()
        i += 1 if count else 0
    u = half_step(dt)
    return y, (d + 16) * 2.0 ** -24 * (1 + u) * mag + u * y.abs() + tiny(dt)


def table(rows, rot, device, base=10000.0):
    freq = base ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    angle = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()


def starts(lengths, device):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)


def check(got, want, bound):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)  # a NaN is bad
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside the bound; first at "
                           f"{bad.nonzero()[0].tolist()}: {got[tuple(bad.nonzero()[0])]} for "
                           f"{want[tuple(bad.nonzero()[0])]} +- {bound[tuple(bad.nonzero()[0])]}")
