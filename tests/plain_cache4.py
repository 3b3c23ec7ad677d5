"""The 4-bit cache and attention over it, plainly and in 64 bits (NumPy, token by token): what the GPU tests compare with."""
import numpy as np
import torch


def bf16(x):
    return torch.as_tensor(np.asarray(x, dtype=np.float64)).float().bfloat16().double().numpy()


def bf16_bits(x):
    return int(torch.tensor(float(x), dtype=torch.float32).bfloat16().view(torch.int16).item()) & 0xFFFF


def encode(x):
    """One vector -> (codes, step, low); low is never -0."""
    x = np.asarray(x, dtype=np.float64)
    if not np.isfinite(x).all() or abs(x.max() - bf16(x.min())) > np.finfo(np.float32).max:
        return np.zeros(len(x), dtype=int), float("nan"), float(bf16(np.nanmin(x)))
    low = float(bf16(x.min())) + 0.0
    step = float(bf16(np.float32((x.max() - low) / 15.0)))
    if step <= 0.0:      # (below 0: low was rounded above the highest entry)
        return np.zeros(len(x), dtype=int), 0.0, low
    return np.clip(np.rint((x - low) / step), 0, 15).astype(int), step, low


def halves_of_value(hd, t):
    """The place of every entry of token t's value among a tile's half bytes: words of four entries of two tokens, a group of
    four tokens after another, sixteen chunks of hd / 16 entries in each."""
    C, four, pair, odd, out = hd // 16, t // 4, (t // 2) % 2, t % 2, []
    for d in range(hd):
        word0 = (four * 16 + d // C) * (C // 2)
        if C == 2:
            out.append(8 * word0 + 2 * (2 * odd + pair) + d % 2)
        else:
            out.append(8 * (word0 + pair * (C // 4) + (d % C) // 4) + 4 * odd + d % 4)
    return np.array(out)


def write(cache, slot, kvh, key, value):
    """Token ``slot``'s key and value into cache [pages, nkv, tiles, bytes] (NumPy uint8)."""
    hd, page = len(key), 16 * cache.shape[2]
    tile, t = cache[slot // page, kvh, slot % page // 16], slot % 16
    for x, at, places in ((key, 0, t * hd + np.arange(hd)), (value, 8 * hd + 64, halves_of_value(hd, t))):
        codes, step, low = encode(x)
        for c, n in zip(codes, places):
            b = at + n // 2
            tile[b] = (tile[b] & 0x0F | c << 4) if n % 2 else (tile[b] & 0xF0 | c)
        if np.isnan(step):
            tile[at + 8 * hd + 4 * t:][:2] = np.frombuffer(np.uint16(0x7FC0).tobytes(), dtype=np.uint8)
        else:
            tile[at + 8 * hd + 4 * t:][:2] = np.frombuffer(np.uint16(bf16_bits(step)).tobytes(), dtype=np.uint8)
        tile[at + 8 * hd + 4 * t + 2:][:2] = np.frombuffer(np.uint16(bf16_bits(low)).tobytes(), dtype=np.uint8)


def parts(cache, nkv, hd):
    """All tokens of a cache (torch uint8, any device) -> (k codes, k step, k low, v codes, v step, v low), codes [slots, nkv, hd]
    and the others [slots, nkv, 1], float64."""
    pages, _, tiles, _ = cache.shape
    out = []
    for at, values in ((0, False), (8 * hd + 64, True)):
        b = cache[..., at:at + 8 * hd]
        halves = torch.stack([b & 15, b >> 4], -1).flatten(-2)
        if values:
            where = np.concatenate([halves_of_value(hd, t) for t in range(16)])
            halves = halves[..., torch.as_tensor(where, device=cache.device)]
        pair = cache[..., at + 8 * hd:at + 8 * hd + 64].contiguous().view(torch.bfloat16).view(pages, nkv, tiles, 16, 2).double()
        shaped = lambda x: x.permute(0, 2, 3, 1, 4).reshape(pages * tiles * 16, nkv, -1)
        out += [shaped(halves.view(pages, nkv, tiles, 16, hd).double()), shaped(pair[..., :1]), shaped(pair[..., 1:])]
    return out


def attend(q, held, slots_of, visible, nh, nkv, scale, dtype):
    """q [rows, nh, hd] float64; slots_of[r]: the slots of row r's sequence (tokens 0 ..); visible[r]: (first, end) of what row r sees.
    -> (out, tol) [rows, nh, hd]: the result in 64 bits, and how far a kernel may be from it.

    The tolerance, term by term (u = 2^-24, and sums of n products in 32 bits taken as 16 u of the sum of their magnitudes, what a
    tree of matrix instructions and a walk over partial sums with a few dozen roundings stay below; B = 128 for bfloat16, 16 for float;
    mid = low + 8 step):
      score      q . k is formed as step * (q . (B + c) - (B + 8) * sum q) + mid * sum q: off by e = 16 u * scale * sum|q| *
                 ((B + 16) step + |mid|) of the largest token, plus u |s| * 4 for the multiplications behind it; a score's error moves p
                 by twice itself, and the hardware's exp2 adds 2 u |s| + 2 u
      output     sum of p step (B + c) less B + 8 of sum (p step), plus sum of p mid: 16 u of sum p ((B + 16) step + |mid|), twice for
                 the division's parts
      bfloat16   p * step is rounded (2^-8 of it at most, what it is multiplied with is c - 8), and so is the output (2^-8 of it)."""
    kc, ks, kl, vc, vs, vl = held
    u, w = 2.0 ** -24, 144.0 if dtype == torch.bfloat16 else 32.0
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for r in range(q.shape[0]):
        first, end = visible[r]
        if end <= first:
            continue
        s = slots_of[r][first:end]
        for h in range(nh):
            g = h * nkv // nh
            k, v = kl[s, g] + ks[s, g] * kc[s, g], vl[s, g] + vs[s, g] * vc[s, g]
            x = (k @ q[r, h]) * scale
            p = torch.softmax(x, 0)
            out[r, h] = p @ v
            k_mid, v_mid = (kl[s, g] + 8 * ks[s, g]).abs(), (vl[s, g] + 8 * vs[s, g]).abs()
            e = 16 * u * abs(scale) * q[r, h].abs().sum() * (w * ks[s, g] + k_mid).max() + 8 * u * x.abs().max() + 4 * u
            t = 2 * e * (p @ (v - out[r, h]).abs()) + 2 * 16 * u * (p @ (w * vs[s, g] + v_mid + 0 * v))
            if dtype == torch.bfloat16:
                t = t + 2.0 ** -8 * (p @ (vs[s, g] * (vc[s, g] - 8).abs())) + 2.0 ** -8 * out[r, h].abs()
            tol[r, h] = t
    return out, tol
