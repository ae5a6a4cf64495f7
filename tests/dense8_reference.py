"""The 8-bit dense layer from its definition, in 64 bits on the CPU (test infrastructure)."""
import torch

BLADES = {1: (0,), 2: (0, 1), 4: (0, 1, 2, 3), 8: (0, 1, 2, 4, 3, 5, 6, 7)}


def terms(dim):
    """(l, r, d, sign) of the product of components: l of the input, r of the filter, d of the output."""
    out = []
    for l in range(dim):
        for r in range(dim):
            if dim == 8:                                 # GA(3,0,0): blades as sets of generators, all squares +1
                a, b = BLADES[8][l], BLADES[8][r]
                swaps = sum(bin((a >> s) & b).count("1") for s in (1, 2))
                out.append((l, r, BLADES[8].index(a ^ b), -1.0 if swaps & 1 else 1.0))
            else:                                        # i^2 = j^2 = k^2 = -1, ij = k, jk = i, ki = j
                negative = l and r and (l == r or (dim == 4 and (l, r) in ((2, 1), (3, 2), (1, 3))))
                out.append((l, r, l ^ r, -1.0 if negative else 1.0))
    return out


def e4m3(v):
    """float64 of magnitude 448 at most -> the nearest e4m3 number, ties to even."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=-6) - 3)
    return torch.round(v / step) * step


def quantized(x, rows, cols):
    """float64 [D, R, C] rounded in blocks of rows x cols; what is not finite becomes NaN."""
    out = torch.empty_like(x)
    for r in range(0, x.shape[1], rows):
        for c in range(0, x.shape[2], cols):
            block = x[:, r:r + rows, c:c + cols]
            finite = torch.isfinite(block)
            top = torch.where(finite, block, torch.zeros_like(block)).abs().amax(dim=(1, 2), keepdim=True)
            e = torch.zeros_like(top)
            for d in range(top.shape[0]):
                t = float(top[d])
                if t > 0.0:
                    k = -126
                    while 448.0 * 2.0 ** k < t:
                        k += 1
                    e[d] = k
            scale = torch.ldexp(torch.ones_like(top), e)
            out[:, r:r + rows, c:c + cols] = torch.where(finite, e4m3(torch.where(finite, block, torch.zeros_like(block)) / scale) * scale,
                                                         torch.full_like(block, float("nan")))
    return out


def product(dim, a, b):
    """sum of sign * a[l] @ b[r] into component d, and the same of the absolute values."""
    out = torch.zeros((dim, a.shape[1], b.shape[2]), dtype=torch.float64)
    size = torch.zeros_like(out)
    for l, r, d, sign in terms(dim):
        out[d] += sign * (a[l] @ b[r])
        size[d] += a[l].abs() @ b[r].abs()
    return out, size


def rows_by_128(x):
    """Blocks of 1 x 128, one row at a time (the loop over blocks takes the maximum over a whole block)."""
    flat = x.reshape(-1, 1, x.shape[2])
    return quantized(flat, 1, 128).reshape(x.shape)


def cols_by_128(x):
    return rows_by_128(x.transpose(1, 2).contiguous()).transpose(1, 2).contiguous()


def forward(dim, x, w_io, bias=None):
    """x [D, B, I], w_io [D, I, O] as the filter's 8-bit form holds it -> y, sum of |products|."""
    y, size = product(dim, rows_by_128(x), w_io)
    return (y if bias is None else y + bias[:, None, :]), size


def backward(dim, x, w_io, dy):
    """-> dx, its sum of |products|, dw, its sum of |products|"""
    dyr, dyc, xc = rows_by_128(dy), cols_by_128(dy), cols_by_128(x)
    dx, sx = torch.zeros_like(x), torch.zeros_like(x)
    dw, sw = torch.zeros_like(w_io), torch.zeros_like(w_io)
    for l, r, d, sign in terms(dim):
        dx[l] += sign * (dyr[d] @ w_io[r].t())
        sx[l] += dyr[d].abs() @ w_io[r].abs().t()
        dw[r] += sign * (xc[l].t() @ dyc[d])
        sw[r] += xc[l].abs().t() @ dyc[d].abs()
    return dx, sx, dw, sw


def bound(value, size, summed, dtype):
    """How far a result may be off. Products of e4m3 numbers are exact in 8 bits; a sum of `summed` of them goes through summed / 32 additions into
    an fp32 accumulator, each behind an aligned sum of 32 products: every step loses at most a unit in the last place (2^-23) of a partial sum, which the sum
    of the absolute products bounds. One rounding to the result's type follows, half a step relative to the value, or half the smallest number."""
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    acc = (summed / 32 + 32) * 2.0 ** -23 * size
    return acc + half * (value.abs() + acc) + tiny
