"""Plain 64-bit forms of the bucketed and 8-bit operators, and error bounds (no product code).

Bounds: a product of two numbers of 16 or 8 bits is exact in fp32.  A sum of n terms in fp32 is off by at most about
n * u * sum |term| whatever its order, u = 2^-24 where every addition rounds to nearest, 2^-23 where it cuts off, as a tensor
core's adders may.  `sum_bound` takes 2^-23.  One rounding to the output's type adds eps / 2 of the result, or half a step
of its subnormal numbers.
"""

import torch

U = 2.0**-23


def rounding(t, dtype):
    return t.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def sum_bound(magnitude, terms):
    return (terms + 4) * U * magnitude


def close(ours, ref, magnitude, terms, what):
    """ours (any float type) against ref (64 bits), summed over `terms` terms whose sizes add up to `magnitude`."""
    assert ours.shape == ref.shape, what
    if not ref.numel():
        return
    off = (ours.detach().cpu().double() - ref).abs()
    acc = sum_bound(magnitude, terms)
    bound = acc + rounding(ref.abs() + acc, ours.dtype)
    assert torch.isfinite(ours.detach()).all(), f"{what}: not finite"
    worst = (off - bound).max()
    assert worst <= 0, f"{what}: {float(off.flatten()[(off - bound).argmax()]):.3e} off, allowed {float(bound.flatten()[(off - bound).argmax()]):.3e}"


def plan_ref(bucket, count):
    key = torch.where((bucket < 0) | (bucket >= count), torch.full_like(bucket, count), bucket)
    order = torch.sort(key, stable=True).indices
    offsets = torch.tensor([int((key < e).sum()) for e in range(count)] + [int((key < count).sum())])
    return order.to(torch.int32), offsets.to(torch.int32)


def linear_ref(x, w, bias, bucket, count, dy=None):
    """y and, with dy, (dx, dw, dbias), each as (value, sum of the terms' sizes, terms), in 64 bits on the CPU."""
    x, w = x.detach().cpu().double(), w.detach().cpu().double()
    T, K = x.shape
    w = w.reshape(count, -1, K)
    N = w.shape[1]
    b = torch.zeros(count, N, dtype=torch.float64) if bias is None else bias.detach().cpu().double().view(count, N)
    y, ym = torch.zeros(T, N).double(), torch.zeros(T, N).double()
    dx, dxm = torch.zeros(T, K).double(), torch.zeros(T, K).double()
    dw, dwm = torch.zeros_like(w), torch.zeros_like(w)
    db, dbm = torch.zeros_like(b), torch.zeros_like(b)
    most = 0
    for e in range(count):
        r = torch.nonzero(bucket.cpu() == e).view(-1)
        most = max(most, len(r))
        y[r] = x[r] @ w[e].T + b[e]
        ym[r] = x[r].abs() @ w[e].abs().T + b[e].abs()
        if dy is not None:
            g = dy.detach().cpu().double()[r]
            dx[r], dxm[r] = g @ w[e], g.abs() @ w[e].abs()
            dw[e], dwm[e] = g.T @ x[r], g.abs().T @ x[r].abs()
            db[e], dbm[e] = g.sum(0), g.abs().sum(0)
    out = {"y": (y, ym, K)}
    if dy is not None:
        out |= {"dx": (dx, dxm, N), "dw": (dw.view(-1, K), dwm.view(-1, K), most), "db": (db.view(-1), dbm.view(-1), most)}
    return out


MAX8 = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def scale_ref(block, format):
    """Scale of one block by its definition, in 64 bits."""
    v = block.double()
    a = float(v[torch.isfinite(v)].abs().max()) if torch.isfinite(v).any() else 0.0
    if a == 0.0:
        return 1.0
    k = -126
    while 2.0**k * MAX8[format] < a:
        k += 1
    return 2.0**k


def quantize_ref(m, block_rows, format):
    """(q as fp32 values, scale) of one matrix in blocks of block_rows x 128, by torch's own conversion of v / scale."""
    rows, K = m.shape
    R, C = -(-rows // block_rows), -(-K // 128)
    q, s = torch.empty(rows, K), torch.empty(R, C)
    for r in range(R):
        for c in range(C):
            blk = m[r * block_rows : (r + 1) * block_rows, c * 128 : (c + 1) * 128].float()
            s[r, c] = scale_ref(blk, format)
            q[r * block_rows : (r + 1) * block_rows, c * 128 : (c + 1) * 128] = (blk.double() / s[r, c].double()).float().to(format).float()
    return q, s
