"""The 4-bit KV page format and its attention in 64 bits, without the framework's code."""
import numpy as np
import torch

GROUP = 64


def quantise(x):
    """float64 [..., hd] -> (codes [..., hd] 0..15, scale [..., groups], zero [..., groups])."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = np.maximum(g.max(-1), 0), np.minimum(g.min(-1), 0)
    m, e = np.frexp((hi - lo) / 15)
    scale = np.ldexp(np.ceil(m * 16) / 16, e)
    scale = np.where((hi - lo) / 15 < 2.0 ** -126, 0.0, scale)
    safe = np.where(scale > 0, scale, 1.0)
    zero = np.where(scale > 0, np.rint(-lo / safe), 0)
    codes = np.where(scale[..., None] > 0, np.minimum(15, np.rint(g / safe[..., None]) + zero[..., None]), 0)
    return codes.reshape(x.shape), scale, zero


def unpack(codes, words):
    """Page tensors -> (codes, scale, zero) as float64 arrays."""
    c = codes.cpu().numpy()
    out = np.empty((*c.shape[:-1], 2 * c.shape[-1]))
    out[..., 0::2], out[..., 1::2] = c % 16, c // 16
    w = words.cpu().numpy().astype(np.int64)
    e, m = (w >> 7) % 256, (w >> 4) % 8
    return out, np.where(e > 0, np.ldexp(1 + m / 8, e - 127), 0.0), (w % 16).astype(np.float64)


def values(codes, words):
    c, s, z = unpack(codes, words)
    s, z = np.repeat(s, GROUP, -1), np.repeat(z, GROUP, -1)
    return torch.from_numpy(s * (c - z))


def random_pages(blocks, nkv, bs, hd, seed, device="cpu", scale=1.0):
    """Codes and words of plausible content, made without quantising anything."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (blocks, nkv, bs, hd // 2), generator=g, dtype=torch.int64).to(torch.uint8)
    s = (0.05 + 0.3 * torch.rand(blocks, nkv, bs, hd // GROUP, generator=g)) * scale
    words = (s.bfloat16().view(torch.int16).int() & 0x7FF0) | torch.randint(4, 12, s.shape, generator=g).int()
    return codes.to(device), words.to(torch.int16).to(device)


def attention(q, k_pages, v_pages, cu, lens, tables, scale):
    """(output, sum of p |v| per output) in float64; rows that see no key give zeros."""
    q = q.double().cpu()
    k, v = values(*k_pages), values(*v_pages)
    nblk, nkv, bs, hd = k.shape
    T, nh, _ = q.shape
    out, mag = torch.zeros(T, nh, hd, dtype=torch.float64), torch.zeros(T, nh, hd, dtype=torch.float64)
    tables = tables.cpu()
    for i in range(len(lens)):
        lo, hi = cu[i], cu[i + 1]
        n = min(lens[i], tables.shape[1] * bs)
        if hi == lo or n <= 0:
            continue
        ids = tables[i, :-(-n // bs)].long()
        ok = ((ids >= 0) & (ids < nblk)).repeat_interleave(bs)[:n]
        ids = ids.clamp(0, nblk - 1)
        ks, vs = (x[ids].transpose(1, 2).reshape(-1, nkv, hd)[:n] for x in (k, v))
        last = torch.arange(lens[i] - (hi - lo), lens[i])[:, None]
        sees = (torch.arange(n)[None] <= last) & ok
        any_row = sees.any(1)
        for h in range(nh):
            a = (q[lo:hi, h] @ ks[:, h // (nh // nkv)].T) * scale
            a = torch.softmax(a.masked_fill(~sees, -torch.inf), -1)
            a[~any_row] = 0
            vh = torch.where(ok[:, None], vs[:, h // (nh // nkv)], 0.0)
            out[lo:hi, h], mag[lo:hi, h] = a @ vh, a @ vh.abs()
    return out, mag


def attention_tolerance(out, mag):
    """The weight of each value is rounded to bfloat16 once (off by 2^-8 of itself at most), the output
    once more (2^-8 of itself); scores and sums in fp32 stay within 2^-12 of the magnitudes summed."""
    return 2.0 ** -8 * (out.abs() + mag) + 2.0 ** -12 * mag + 1e-30
