"""The definition of dense8_reference.py without loops over blocks, for large layers and any device (test infrastructure)."""
import torch

import dense8_reference as ref


def quantized(x, rows, cols):
    """float64 [D, R, C] rounded in blocks of rows x cols; what is not finite becomes NaN."""
    d, r, c = x.shape
    padded = torch.zeros((d, -(-r // rows) * rows, -(-c // cols) * cols), dtype=x.dtype, device=x.device)
    padded[:, :r, :c] = x
    blocks = padded.view(d, padded.shape[1] // rows, rows, padded.shape[2] // cols, cols)
    finite = torch.isfinite(blocks)
    kept = torch.where(finite, blocks, torch.zeros_like(blocks))
    top = kept.abs().amax(dim=(2, 4), keepdim=True)
    m, e = torch.frexp(top)                                  # top = m * 2^e, m in [1/2, 1); 448 = 7/8 * 2^9
    e = torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=-126)
    scale = torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, torch.zeros_like(e)))
    out = torch.where(finite, ref.e4m3(kept / scale) * scale, torch.full_like(kept, float("nan")))
    return out.view(padded.shape)[:, :r, :c].contiguous()


def by_rows(x):
    return quantized(x, 1, 128)


def by_cols(x):
    return quantized(x, 128, 1)


def forward(dim, x, w_io):
    """x [D, B, I], w_io [D, I, O] as the filter's 8-bit form holds it -> y, sum of |products|."""
    xr = by_rows(x)
    y = torch.zeros((dim, x.shape[1], w_io.shape[2]), dtype=x.dtype, device=x.device)
    size = torch.zeros_like(y)
    for l, r, d, sign in ref.terms(dim):
        y[d] += sign * (xr[l] @ w_io[r])
        size[d] += xr[l].abs() @ w_io[r].abs()
    return y, size


def backward(dim, x, w_io, dy):
    """-> dx, its sum of |products|, dw, its sum of |products|"""
    dyr, dyc, xc = by_rows(dy), by_cols(dy), by_cols(x)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w_io)
    sx, sw = torch.zeros_like(x), torch.zeros_like(w_io)
    for l, r, d, sign in ref.terms(dim):
        dx[l] += sign * (dyr[d] @ w_io[r].t())
        sx[l] += dyr[d].abs() @ w_io[r].abs().t()
        dw[r] += sign * (xc[l].t() @ dyc[d])
        sw[r] += xc[l].abs().t() @ dyc[d].abs()
    return dx, sx, dw, sw
