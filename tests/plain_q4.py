"""The cache in 4 bits in plain float64: rows to codes and back, pages, attention over them (csrc/cuda/q4.cuh has the layout)."""
import math

import torch

# nibble of element e of a 32-bit word of codes
SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]


def page_bytes(page, hd):
    return (page * (hd // 2 + 4) + 15) // 16 * 16


def quantised(x):
    """x [.., hd] (exact in float32) -> codes (int64), scale and zero (bfloat16): the float32 steps of the definition."""
    x = x.float()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, zero = ((high - low) / 15).to(torch.bfloat16), low.to(torch.bfloat16)
    s = scale.float()
    code = torch.where(s > 0, (x - zero.float()) / s, torch.zeros_like(x)).round().clamp(0, 15).long()
    return code, scale, zero


def write(cache, B, page_id, off, x):
    """Row ``off`` of page ``page_id`` (cache uint8 [pages, nkv, bytes], pages of B) <- x [nkv, hd]."""
    nkv, hd = x.shape
    code, scale, zero = quantised(x)
    w = torch.zeros((nkv, hd // 8), dtype=torch.int64)
    for e in range(8):
        w |= code[:, e::8] << SHIFTS[e]
    raw = torch.stack([(w >> (8 * b)) & 255 for b in range(4)], dim=-1).flatten(1).to(torch.uint8)
    cache[page_id, :, off * hd // 2:(off + 1) * hd // 2] = raw
    pair = torch.cat((scale, zero), dim=-1).contiguous().view(torch.uint8)
    cache[page_id, :, B * hd // 2 + 4 * off:B * hd // 2 + 4 * off + 4] = pair


def read(cache, hd, B):
    """Values float64 [pages, nkv, B, hd] of a whole cache."""
    pages, nkv, _ = cache.shape
    n = B * hd // 2
    raw = cache[..., :n].reshape(pages, nkv, B, hd // 8, 4).long()
    w = sum(raw[..., b] << (8 * b) for b in range(4))
    code = torch.stack([(w >> s) & 15 for s in SHIFTS], dim=-1).flatten(-2).double()
    pair = cache[..., n:n + 4 * B].contiguous().view(torch.bfloat16).double().view(pages, nkv, B, 2)
    return pair[..., 1:] + pair[..., :1] * code


def rotated(x, cos, sin, interleaved):
    """x [T, heads, hd], cos and sin [T, rotary/2]: in the type of x, product by product."""
    r = 2 * cos.shape[1]
    y = x.clone()
    c, s = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    ra, rb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = ra, rb
    else:
        y[..., :r // 2], y[..., r // 2:r] = ra, rb
    return y


def attention(q, k, v, tables, spans, nh, nkv, B, scale, window=0, softcap=0.0, sink=None):
    """q [rows, nh, hd] float64; k, v values of all pages [pages, nkv, B, hd]; spans: (start, rows) a request.  float64 rows."""
    out = torch.zeros_like(q)
    row = 0
    for i, (start, n) in enumerate(spans):
        end = start + n
        ids = tables[i, :(end + B - 1) // B].long()
        K, V = (x[ids].transpose(0, 1).flatten(1, 2)[:, :end] for x in (k, v))
        for r in range(n):
            at = start + r
            lo = max(0, at + 1 - window) if window else 0
            for h in range(nh):
                g = h // (nh // nkv)
                s = K[g, lo:at + 1] @ q[row, h] * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if sink is not None:
                    s = torch.cat((s, sink[h].double().reshape(1)))
                p = torch.softmax(s, 0)[:at + 1 - lo]
                out[row, h] = p @ V[g, lo:at + 1]
            row += 1
    return out
