"""The FP8 operators by their definition, in 64 bits, and how far a kernel's result may be from it.

A product's tolerance.  Codes are exact, products of two e4m3 values too; what is rounded is
  * every addition, off by at most 2^-23 (an addition that truncates) of the absolute sum S = sum_k |x w| it adds to.  Kernels that
    scale every K block's sum in fp32: at most 128 additions inside a block and one per block outside; the product of the two scales
    and the product with it are off by 3 * 2^-24 of S at most.  Kernels that leave the scales to the tensor core: each of the K / 32 MMAs
    adds to one accumulator, and inside an MMA 32 products meet, whose roundings are relative to that MMA's share of S.  So
    128 + K / 32 + 2 covers both,
  * the result to its 16-bit type: half a step, 2^-8 (bf16) or 2^-11 (fp16) of its value, and 2^-25 absolutely where fp16 has
    subnormals (bf16's lie below everything here).
So |y - exact| <= (128 + K / 32 + 2) 2^-23 S + half * (|exact| + that) + 2^-25.
"""
import numpy as np
import torch

BLOCK = 128
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ceil_div(a, b):
    return -(-a // b)


def pow2(e):
    """2^e as float64, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def scale_values(s):
    if s.dtype == torch.float8_e8m0fnu:
        b = s.view(torch.uint8).to(torch.int64)
        return torch.where(b == 255, torch.full(b.shape, float("nan"), dtype=torch.float64, device=s.device), pow2(b - 127))
    return s.double()


def row_values(q, s):
    """Codes [M, K] times their scales [M, blocks]."""
    return q.double() * scale_values(s).repeat_interleave(BLOCK, dim=-1)[..., :q.shape[-1]]


def weight_values(q, s):
    v = scale_values(s).repeat_interleave(BLOCK, dim=-1)[..., :q.shape[-1]].repeat_interleave(BLOCK, dim=-2)
    return q.double() * v[..., :q.shape[-2], :]


def block_exponent(a):
    """The smallest e with a <= 448 * 2^e, at least -126; 0 for a = 0.  a float64 (exact values of narrower types)."""
    m, ex = torch.frexp(a)
    e = torch.where(m > 0.875, ex - 8, ex - 9).clamp(min=-126)
    return torch.where(a > 0, e, torch.zeros_like(e))


def round_e4m3(t):
    """float64 values of magnitude at most 448 to the nearest e4m3 value, ties to even."""
    _, ex = torch.frexp(t)
    step = pow2((ex - 1).clamp(min=-6) - 3)
    return torch.round(t / step) * step


def quantise(x, rows=1):
    """(values of the codes, exponents of the scales) of x [M, K] with one scale per `rows` rows and 128 columns; NaN for a block that is
    not finite."""
    M, K = x.shape
    mb, kb = ceil_div(M, rows), ceil_div(K, BLOCK)
    p = torch.zeros(mb * rows, kb * BLOCK, dtype=torch.float64, device=x.device)
    p[:M, :K] = x.double()
    b = p.view(mb, rows, kb, BLOCK)
    a = b.abs().amax(dim=(1, 3))
    bad = ~torch.isfinite(a)
    e = block_exponent(torch.where(bad, torch.zeros_like(a), a))
    q = round_e4m3(torch.where(bad[:, None, :, None], torch.zeros_like(b), b) / pow2(e)[:, None, :, None])
    q = torch.where(bad[:, None, :, None], torch.full_like(q, float("nan")), q).reshape(mb * rows, kb * BLOCK)[:M, :K]
    return q, e, bad


def quantised_values(x):
    q, e, bad = quantise(x)
    return q * pow2(e).repeat_interleave(BLOCK, dim=1)[:, :x.shape[1]]


def sum_roundings(K):
    return 128 + ceil_div(K, 32) + 2


def product_tolerance(xv, wv, out_dtype):
    """(exact, tolerance) of xv @ wv.T for values xv [M, K], wv [N, K] in float64."""
    exact = xv @ wv.T
    acc = sum_roundings(xv.shape[1]) * 2.0 ** -23 * (xv.abs() @ wv.abs().T)
    if out_dtype is None:
        return exact, acc
    half = HALF_STEP[out_dtype]
    return exact, acc + half * (exact.abs() + acc) + 2.0 ** -25


def assert_within(y, exact, tol, what=""):
    y = y.double()
    assert y.shape == exact.shape, (what, y.shape, exact.shape)
    nan = torch.isnan(exact)
    assert torch.equal(torch.isnan(y), nan), f"{what}: NaN in other places"
    over = ((y - exact).abs() - tol)[~nan]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} off, worst by {over.max():.3g}"


def random_rows(g, M, K, dtype=torch.float32, scale=1.0):
    x = torch.randn(M, K, generator=g, device="cuda") * scale
    x[:, ::29] *= 6.0
    return x.to(dtype)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def arbitrary_scales(s, g):
    """Scales that are no powers of two, near the given ones."""
    return scale_values(s).float() * (0.75 + 0.5 * torch.rand(s.shape, generator=g, device=s.device))


def route_reference(logits, k, renormalize):
    """numpy, 64 bits: ids, weights, rows, offsets."""
    l = np.asarray(logits, dtype=np.float64)
    T, E = l.shape
    key = np.where(np.isnan(l), np.inf, l)
    big = np.isnan(l)
    ids = np.zeros((T, k), dtype=np.int64)
    weights = np.zeros((T, k))
    for t in range(T):
        order = sorted(range(E), key=lambda e: (not big[t, e], -key[t, e], e))[:k]
        ids[t] = order
        with np.errstate(invalid="ignore"):
            top = l[t, order[0]]
            p = np.exp(l[t] - top)
            chosen = p[order]
            weights[t] = 0.0 if top == -np.inf else chosen / (chosen.sum() if renormalize else p.sum())
    return (ids, weights) + group_reference(ids, E)


def group_reference(ids, E):
    flat = np.asarray(ids).ravel()
    rows = np.full(flat.shape, -1, dtype=np.int64)
    offsets, at = [0], 0
    for e in range(E):
        mine = np.nonzero(flat == e)[0]
        rows[mine] = at + np.arange(len(mine))
        at += len(mine)
        offsets.append(at)
    return rows.reshape(np.shape(ids)), np.array(offsets)
