"""Plain forms, in 64 bits and on the CPU, of the operators on 4-bit weights and sorted tokens, with bounds on what FP32 sums may be off."""
import torch

import synth

pkg = synth.pkg


def up(n, m):
    return (n + m - 1) // m * m


def make(rng, rows, cols, group, count=None, spread=0.2, scale=0.0075):
    """Random codes of all sixteen values and scales; what lies behind the last column and group is garbage, NaN among it."""
    lead = () if count is None else (count,)
    groups = -(-cols // group)
    codes = torch.randint(0, 256, lead + (rows, up(cols, 32) // 2), generator=rng, dtype=torch.int32).to(torch.uint8)
    scales = torch.full(lead + (rows, up(groups, 8)), float("nan"), dtype=torch.bfloat16)
    scales[..., :groups] = (scale * torch.exp(spread * torch.randn(lead + (rows, groups), generator=rng))).to(torch.bfloat16)
    return codes, scales


def values(codes, scales, cols, group):
    """W in FP64."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :cols].double() - 8.0
    return c * scales.double().repeat_interleave(group, -1)[..., :cols]


def handle(codes, scales, rows, cols, group):
    return pkg.W4(codes.cuda(), scales.cuda(), rows, cols, group)


# What a product may be off. Additions: each is off by at most 2^-23 of the partial sum (the tensor cores cut, elsewhere half of
# it); a matrix instruction takes 16 columns with at most two such cuts (or is exact in integers), and each group of 32 columns is one
# more addition: at most cols / 16 * 2 + cols / 32 + 16 in a row, whatever order they are taken in; a partial sum is at most the sum of
# |w_k x_k|. Activations: fixed-point numbers of 22 bits (BF16 rows: 14) below the power of two over the largest of their 128
# columns, off by half a step, 2^-23 (2^-15) of that power, so 2^-22 (2^-14) of the largest; or floating ones of 22 bits, off by less
# (BF16: exact). `own` adds what one F16 term is off, 2^-12 of the value.
def product_bound(w, x, f32=True, own=0.0):
    cols = x.shape[-1]
    steps = 2 * (cols // 16 + 1) + cols // 32 + 16
    block = torch.nn.functional.pad(x.abs(), (0, up(cols, 128) - cols)).view(x.shape[0], -1, 128).amax(2).repeat_interleave(128, 1)[:, :cols]
    held = block * (2.0 ** -22 if f32 else 2.0 ** -14) + x.abs() * own
    return (x.abs() @ w.abs().t()) * (steps * 2.0 ** -23) + held @ w.abs().t()


def rounded(y, dtype):
    """What rounding to the output's type may add."""
    return y.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).tiny


def swiglu(g, u, limit):
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(g) * u


def experts(x, idx, weights, gate, up_, down, limit, f32):
    """(out, bound) of the routed experts; gate, up_, down: FP64 values [E][..][..]."""
    T, K = idx.shape
    out, off = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        for k in range(K):
            e = int(idx[t, k])
            if not 0 <= e < gate.shape[0]:
                continue
            row = x[t:t + 1]
            g, u = row @ gate[e].t(), row @ up_[e].t()
            eg, eu = product_bound(gate[e], row, f32), product_bound(up_[e], row, f32)
            h = swiglu(g, u, limit)
            cu = u.abs().clamp(max=limit) + eu
            # |d silu / d g| <= 1.1 where the clamp lets it through; the sigmoid is 1.53 units of 2^-23 off, two products round
            eh = 1.1 * cu * eg + (g.clamp(max=limit) * torch.sigmoid(g.clamp(max=limit))).abs() * eu + h.abs() * 3 * 2.0 ** -23
            y = h @ down[e].t()
            ey = eh @ down[e].abs().t() + product_bound(down[e], h.abs() + eh, f32, 0.0 if f32 else 2.0 ** -12)
            wt = float(weights[t, k])
            out[t] += wt * y[0]
            # the sum over the picks: one rounding each, of a partial sum that is no larger than the sum of magnitudes
            off[t] += abs(wt) * (ey[0] + K * 2.0 ** -24 * (y[0].abs() + ey[0]))
    return out, off
