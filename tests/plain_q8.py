"""The cache in 8 bits in plain operations (csrc/cuda/q8.cuh has the format), attention over it and over rows, and how far each kernel may be off.

Codes are compared bit by bit: kernel and definition take the same float32 steps with IEEE roundings.

Attention, element by element, with probabilities p_j (sum 1), values v_j, o = sum p_j v_j, half a step of each rounding:
 * the result: 2^-8 |o| (bfloat16), 2^-24 |o| (float32).
 * weights, rounded once where they enter a product: ``weight`` * sum p |v| (float16 2^-11, bfloat16 2^-8); where a row's maximum is
   renewed inside a tile of 128 keys, weights of up to three pieces of 32 are rounded again: four times that.  float16 weights below
   2^-14 of their unit, which is at most 2^13 below the largest weight's next power of two or at most it, are off by up to 2^-25 of the
   unit: 2^-24 max(p scale) sum |code|.
 * sums in float32 and exponentials: 2^-24 times the number of additions a term goes through (at most keys + 16) of sum p |v|, and
   ``exponential`` of the same (2^-21 for ex2.approx and the arithmetic around it).
 * scores that are off by e_j move the result by at most sum p_j e_j (|v_j| + |o|): e = (hd + 8) 2^-24 sum |q k| scale + 8 * 2^-24 (1 + |score|);
   q as float16 times a power of two (pages): elements below 2^-29 of the row's largest are off by 2^-39 of it, e += 2^-39 max|q| sum |k| scale;
   tanh (capped scores): 2^-20 cap.
"""
import torch

FP8 = torch.float8_e4m3fn
LEAST = -60


def scale_for(largest):
    """float32: the least 2^e, e >= -60, with 448 * 2^e >= largest."""
    f, e = torch.frexp(largest)
    e = torch.where(f > 0.875, e - 8, e - 9)
    e = torch.where(largest > 0, e, torch.full_like(e, LEAST)).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(largest), e)


def coded(x, scale):
    """Codes (uint8) of float32 x over a scale; not-a-number for what is not finite."""
    y = x / scale
    return torch.where(torch.isfinite(x), y, torch.full_like(y, float("nan"))).to(FP8).view(torch.uint8)


def values(codes, scale):
    """float32 [pages, nkv, B, hd] of codes (uint8) and scales [pages, nkv]."""
    return codes.view(FP8).float() * scale[..., None, None]


def write(codes, scale, slots, rows):
    """Rows float32 [T, nkv, hd] into their slots: codes uint8 [pages, nkv, B, hd] and scale [pages, nkv], page by page."""
    pages, nkv, B, hd = codes.shape
    by_page = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * B:
            by_page.setdefault(s // B, []).append((t, s % B))
    for page, here in by_page.items():
        x = rows[[t for t, _ in here]]                                     # [n, nkv, hd]
        size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((0, 2))
        need, old = scale_for(size), scale[page].clone()
        anew = any(off == 0 for _, off in here)
        new = need if anew else torch.maximum(need, old)
        if not anew:
            for h in range(nkv):
                if old[h] < new[h]:
                    codes[page, h] = coded(codes[page, h].view(FP8).float() * (old[h] / new[h]), torch.ones(()))
        scale[page] = new
        for i, (_, off) in enumerate(here):
            codes[page, :, off] = coded(x[i], new[:, None])


def pool(pages, nkv, B, hd, seed, size=1.0, spread=0):
    """A pool of quantised normal rows on the CPU, pages of sizes 2^0 .. 2^spread apart."""
    g = torch.Generator().manual_seed(seed)
    x = size * torch.randn((pages, nkv, B, hd), generator=g) * 2.0 ** torch.randint(0, spread + 1, (pages, nkv, 1, 1), generator=g).float()
    scale = scale_for(x.abs().amax((-1, -2)))
    return coded(x, scale[..., None, None]), scale


def gathered(codes, scale, table, keys):
    """float64 [nkv, keys, hd] of a request's pages."""
    B = codes.shape[2]
    ids = table[:-(-keys // B)].long()
    return values(codes[ids], scale[ids]).double().transpose(0, 1).flatten(1, 2)[:, :keys]


KINDS = {"single": dict(weight=2.0 ** -11, small=True, result=2.0 ** -8, half=True),
         "portion": dict(weight=4 * 2.0 ** -11, small=True, result=2.0 ** -8, half=True),
         "laid out": dict(weight=4 * 2.0 ** -8, small=False, result=2.0 ** -8, half=False),
         "prompt": dict(weight=4 * 2.0 ** -8, small=False, result=2.0 ** -8, half=False),
         "plain bfloat16": dict(weight=0.0, small=False, result=2.0 ** -8, half=False),
         "plain float32": dict(weight=0.0, small=False, result=2.0 ** -24, half=False)}


def attend(kind, q, k, v, at, scale, window=0, softcap=0.0, sink=None, lost=None, exponential=2.0 ** -21):
    """Rows of one request and their room.  q float64 [n, nh, hd], k and v float64 [nkv, keys, hd], positions ``at`` [n];
    ``lost``: (first, last) keys left out (a planted mistake)."""
    c, eps = KINDS[kind], 2.0 ** -24
    n, nh, hd = q.shape
    G, keys = nh // k.shape[0], k.shape[1]
    key = torch.arange(keys)
    seen = key <= at[:, None]
    if window:
        seen = seen & (key > at[:, None] - window)
    if lost is not None:
        seen = seen & ~((key >= lost[0]) & (key < lost[1]))
    want, room = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(nh):
        kk, vv = k[h // G], v[h // G]
        vv0 = torch.where(seen.any(0)[:, None], vv, torch.zeros_like(vv))          # (what nobody sees may be anything)
        kk0 = torch.where(seen.any(0)[:, None], kk, torch.zeros_like(kk))
        s = (q[:, h] @ kk0.T) * scale
        size = (q[:, h].abs() @ kk0.abs().T) * scale
        e = (hd + 8) * eps * size + 8 * eps * (1 + s.abs())
        if c["half"]:
            e = e + 2.0 ** -39 * q[:, h].abs().amax(-1, keepdim=True) * kk0.abs().sum(-1) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
            e = e + 2.0 ** -20 * softcap
        s = s.masked_fill(~seen, -torch.inf)
        full = torch.cat((s, torch.full((n, 1), float(sink[h]), dtype=s.dtype)), 1) if sink is not None else s
        p = torch.nan_to_num(torch.softmax(full, -1))[:, :keys]
        p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
        e = torch.where(seen, e, torch.zeros_like(e))
        o, a = p @ vv0, p @ vv0.abs()
        want[:, h] = o
        r = c["result"] * o.abs() + (c["weight"] + (keys + 16) * eps + exponential) * a + (p * e) @ vv0.abs() + o.abs() * (p * e).sum(-1, keepdim=True)
        if c["small"]:
            # (a weight is p times its page's scale, a code the value over it: their products are p v)
            top = (p[:, :, None] * vv0.abs()).flatten(1).amax(-1, keepdim=True)
            r = r + eps * top * 448 * seen.sum(-1, keepdim=True)
        room[:, h] = r
    return want, room
