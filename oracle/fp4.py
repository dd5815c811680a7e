"""The microscaled 4-bit operators from their definitions, in 64 bits, on any device.

Independent of the package: quantisation by arithmetic on float64 (every decision exact), the
codes and block scales read back byte by byte from their documented layout.
"""
import math

import torch

BLOCK = {"nv": 16, "mx": 32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def exponent(v):
    """floor(log2 v) for positive float64 v."""
    m, e = torch.frexp(v)
    return e.double() - 1


def e4m3(v):
    """v >= 0 to the nearest E4M3 value, ties to even, at most 448."""
    e = exponent(v.clamp(min=2.0 ** -40)).clamp(min=-6)
    step = torch.pow(torch.full_like(v, 2.0), e - 3)
    return (torch.round(v / step) * step).clamp(max=448.0)


def e2m1(v):
    """v >= 0 to the nearest E2M1 value, ties to even, at most 6."""
    step = torch.full_like(v, 0.5)
    step[v >= 2] = 1.0
    step[v >= 4] = 2.0
    return (torch.round(v / step) * step).clamp(max=6.0)


def pow2(e):
    return torch.ldexp(torch.ones_like(e), e.to(torch.int32))


def quantize(x, fmt):
    """(values [M, K], block scales [M, J] with the row scale in them, row scale [M] or None),
    float64; a block with a non-finite value is NaN."""
    n = BLOCK[fmt]
    x = x.double()
    M, K = x.shape
    J = -(-K // n)
    p = torch.zeros(M, J * n, dtype=torch.float64, device=x.device)
    p[:, :K] = x
    p = p.view(M, J, n)
    bad = ~torch.isfinite(p).all(-1)
    a = torch.where(torch.isfinite(p), p.abs(), 0.0)
    top = a.amax(-1)
    row = None
    if fmt == "mx":
        s = pow2((exponent(top.clamp(min=2.0 ** -160)) - 2).clamp(-127, 127))
    else:
        t = top.amax(-1)
        k = exponent(t.clamp(min=2.0 ** -160) / 2688.0)
        k = torch.where(t > 2688.0 * pow2(k), k + 1, k).clamp(min=-100)
        row = torch.where(t > 0, pow2(k), 1.0)
        s = e4m3(top / (6 * row[:, None])) * row[:, None]
    v = e2m1(a / torch.where(s > 0, s, 1.0)[..., None]) * torch.sign(p.nan_to_num(0.0)) * s[..., None]
    v = torch.where(bad[..., None], math.nan, v)
    return v.reshape(M, -1)[:, :K], torch.where(bad, math.nan, s), row


def values(q):
    """The values an FP4Tensor stands for, read from its bytes."""
    M, K = q.shape
    n = BLOCK[q.fmt]
    codes, scales = q.codes.cpu(), q.scales.cpu()
    k = torch.arange(K)
    c = (codes[:, k // 2].long() >> (4 * (k % 2))) & 15
    v = torch.tensor(E2M1, dtype=torch.float64)[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    J = -(-K // n)
    tiles = -(-J // 4)
    m, j = torch.arange(M)[:, None], torch.arange(J)[None]
    at = (m // 128 * tiles + j // 4) * 512 + m % 32 * 16 + m % 128 // 32 * 4 + j % 4
    b = scales[at].long()
    if q.fmt == "mx":
        s = torch.where(b == 255, math.nan, pow2((b - 127).double()))
    else:
        e, f = b // 8, (b % 8).double()
        s = torch.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * pow2((e - 7).double()))
        s = torch.where(b == 0x7F, math.nan, s)
        if q.row_scale is not None:
            s = s * q.row_scale.cpu().double().reshape(-1, 1)
    return v * s[:, k // n]


def padding(q):
    """(code bytes past K, scale bytes of blocks past the last), which have to be 0."""
    M, K = q.shape
    n = BLOCK[q.fmt]
    codes, scales = q.codes.cpu(), q.scales.cpu()
    J = -(-K // n)
    tiles = -(-J // 4)
    tail = codes[:, -(-K // 2):]
    odd = codes[:, K // 2] >> 4 if K % 2 else codes[:, :0].reshape(-1)
    m, j = torch.arange(M)[:, None], torch.arange(J, tiles * 4)[None]
    at = (m // 128 * tiles + j // 4) * 512 + m % 32 * 16 + m % 128 // 32 * 4 + j % 4
    return torch.cat((tail.reshape(-1), odd.reshape(-1), scales[at].reshape(-1)))


def gelu_tanh(u):
    return 0.5 * u * (1 + torch.tanh(math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3)))


def norm(v, kind, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def residual_norm(x, y, gate=None, residual_scale=1.0, post_norm=None, post_weight=None,
                  post_bias=None, post_eps=1e-6, norm_kind="layer", weight=None, bias=None,
                  scale=None, shift=None, eps=1e-6):
    d = lambda t: None if t is None else t.double()  # noqa: E731
    z = norm(d(y), post_norm, post_eps)
    if post_weight is not None:
        z = z * d(post_weight)
    if post_bias is not None:
        z = z + d(post_bias)
    if gate is not None:
        z = z * d(gate)
    xn = residual_scale * d(x) + z
    h = norm(xn, norm_kind, eps)
    if weight is not None:
        h = h * d(weight)
    if bias is not None:
        h = h + d(bias)
    if scale is not None:
        h = h * (1 + d(scale))
    if shift is not None:
        h = h + d(shift)
    return xn, h
