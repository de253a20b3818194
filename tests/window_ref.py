"""Plain 64-bit implementations and error bounds for the tests of windowed
attention and of the 8-bit KV cache (torch elementary operations)."""
import math

import torch

D = 128
SCALE = 1.0 / math.sqrt(D)
SCALE_F16 = float(torch.tensor(SCALE).half())  # the decode path's default scale
HALF_STEP = 2.0 ** -11  # rounding to f16, relative


def attention64(q, k, v, pos, window=0, sinks=0, scale=SCALE):
    """q [m, Hq, D] rows at positions pos [m]; k, v [n, Hkv, D]: keys 0 .. n-1.
    Returns (out, bound) in 64 bits: the result and what a kernel that
    computes it in one pass with f16 weights may be off by, per element.

    Bound: a weight is rounded to f16 (half a step, relative 2^-11, or 2^-25
    absolute below f16's normal range, relative to the row's largest weight,
    so at most n 2^-25 max|v| in the quotient); the exponent's error dx gives a
    relative ln2 * dx < dx.  dx: an f32 dot product of 128 terms, each partial
    sum rounded or truncated (2^-23), is off by at most 128 * 2^-23 sum|q k|,
    times the scale; ex2.approx 2^-22; the polynomial exponential 7.6e-5;
    numerator and denominator both carry it, hence the factor 2.  Sums of n
    terms in f32 (2^-23 each, across warps and splits at most 64 in a row of
    partial sums of 16-key products) add 2^-16.  The output is rounded to f16."""
    q, k, v = q.double(), k.double(), v.double()
    m, hq, _ = q.shape
    n, hkv, _ = k.shape
    key = torch.arange(n, device=q.device)
    seen = key[None] <= pos[:, None]
    if window:
        seen &= (key[None] > pos[:, None] - window) | (key[None] < sinks)
    used = seen.any(0)  # rows nobody sees may hold NaN
    k = torch.where(used[:, None, None], k, 0.0)
    v = torch.where(used[:, None, None], v, 0.0)
    out = torch.empty_like(q)
    bound = torch.empty_like(q)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = (q[:, h] @ kh.T) * scale
        s[~seen] = -math.inf
        p = torch.softmax(s, -1)
        o = p @ vh
        far = (q[:, h].abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(-1)  # sum |q k| of the row
        dx = far * 128 * 2.0 ** -23 + 2.0 ** -22 + 7.6e-5
        rel = 2 * dx + HALF_STEP + 2.0 ** -16
        bound[:, h] = (rel[:, None] * (p @ vh.abs()) + HALF_STEP * o.abs() + 2.0 ** -25
                       + seen.sum(-1)[:, None] * 2.0 ** -25 * vh.abs().amax())
        out[:, h] = o
    return out, bound


def check(got, ref, bound):
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"error is {worst:.3f} of its bound (max abs {err.max().item():.2e})"


def normal(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g) * scale


def page_pool(caches, page_size, seed, spare=2, fill=float("nan")):
    """Scatters each [B, Hkv, n, ...] cache into a shuffled page pool [pages,
    Hkv, page_size, ...]; rows past n and spare pages hold `fill`.  Returns
    (pools, table [B, pages per sequence])."""
    B, hkv, n = caches[0].shape[:3]
    per = -(-n // page_size)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * per + spare, generator=g)[: B * per].view(B, per).int().cuda()
    pools = []
    for c in caches:
        pool = torch.full((B * per + spare, hkv, page_size) + c.shape[3:], fill, device="cuda").to(c.dtype)
        for b in range(B):
            for i in range(per):
                part = c[b, :, i * page_size:(i + 1) * page_size]
                pool[int(table[b, i]), :, : part.shape[1]] = part
        pools.append(pool)
    return pools, table


def free_pages(table, page_size, low, sinks):
    """Table with the entries of pages wholly between the sinks and key low[b] set to -1."""
    table = table.clone()
    for b in range(table.shape[0]):
        for i in range(table.shape[1]):
            if (i + 1) * page_size <= low[b] and i * page_size >= sinks:
                table[b, i] = -1
    return table


def quantise64(y):
    """[..., D] -> (e4m3 code values, scale) of the 8-bit cache, in 64 bits."""
    top = y.double().abs().amax(-1)
    x = y.double() * torch.where(top > 0, 448.0 / top, 0.0)[..., None]
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    return torch.round(x / step) * step, top / 448.0


def fp8_cache(seed, *shape, scale=1.0):
    """A random 8-bit cache: codes [..., D] float8_e4m3fn, f32 scales [...]."""
    code, s = quantise64(normal(seed, *shape, scale=scale) * torch.exp(normal(seed + 1, *shape[:-1], 1)))
    return code.float().to(torch.float8_e4m3fn), s.float()


def values(codes, scales):
    """What an 8-bit cache stands for, in 64 bits."""
    return codes.float().double() * scales.double()[..., None]
