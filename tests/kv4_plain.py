"""Plain 64-bit forms of the operators around the 4-bit cache, written from their definitions for the tests: rotary
positions, block tables, storing and reading codes, attention.  Works on CPU tensors as well as on the GPU's."""
import math

import numpy as np


def blocks(tokens, size):
    return -(-tokens // size)


def turns(rotary_dim, base=10000.0, scaling="none", factor=1.0, original=0.0, fast=0.0, slow=0.0):
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    plain = base ** (-2.0 * i / rotary_dim) / (2.0 * np.pi)
    if scaling == "linear":
        return plain / factor, 1.0
    if scaling == "yarn":
        pair = [rotary_dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow)]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rotary_dim - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        return plain / factor * ramp + plain * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "banded":
        keep = np.clip((plain * original - slow) / (fast - slow), 0, 1)
        return plain * keep + plain / factor * (1 - keep), 1.0
    return plain, 1.0


def rope(torch, x, positions, table, amplitude, layout):
    """x [tokens, heads, dim]; the turned rows in 64 bits and, per element, amplitude * (|x1| + |x2|)."""
    r = 2 * table.numel()
    phase = positions.double()[:, None] * table[None, :]
    phase = (phase - phase.round()) * (2 * math.pi)
    c, s = (phase.cos() * amplitude)[:, None, :], (phase.sin() * amplitude)[:, None, :]
    y = x.double().clone()
    size = torch.zeros_like(y)
    one, two = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = y[..., one].clone(), y[..., two].clone()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one] = size[..., two] = (a.abs() + b.abs()) * amplitude
    return y, size


def assign(cached, new, table, free, count, bs, capacity):
    table = table.copy()
    slots, positions, starts = [], [], [0]
    for r, (c, n) in enumerate(zip(cached, new)):
        for b in range(blocks(c, bs), blocks(c + n, bs)):
            count -= 1
            table[r, b] = free[count]
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[r, p // bs] * bs + p % bs)
        starts.append(starts[-1] + n)
    fill = [-1] * (capacity - len(slots))
    return dict(table=table, total=[c + n for c, n in zip(cached, new)], starts=starts, slots=slots + fill, positions=positions + fill, count=[count])


# ---- the cache -----------------------------------------------------------------------------------------------------------
def new_cache(torch, count, heads, bs, dim, seed, device="cuda"):
    """Random codes and parameters that are no numbers: whatever is read without having been written shows.  seed None: zeros."""
    code, params = (count, heads, bs, dim // 2), (count, heads, bs, 2)
    if seed is None:
        make = lambda: torch.zeros(code, dtype=torch.uint8, device=device)  # noqa: E731
    else:
        gen = torch.Generator(device=device).manual_seed(seed)
        make = lambda: torch.randint(0, 256, code, generator=gen, dtype=torch.uint8, device=device)  # noqa: E731
    nan = lambda: torch.full(params, math.nan, dtype=torch.bfloat16, device=device)  # noqa: E731
    return dict(k_codes=make(), v_codes=make(), k_params=nan(), v_params=nan())


def bind(B, cache, bs):
    count, heads, _, half = cache["k_codes"].shape
    return B.kv4_cache(blocks=count, block_size=bs, kv_heads=heads, head_dim=2 * half, **cache)


def _eight_bits(torch, x, rounded):
    """x to eight significant bits with `rounded` (floor or ceil), exponents of the normal range."""
    m, e = torch.frexp(x)
    e = torch.maximum(e, torch.full_like(e, -125))          # below 2^-126 BF16 numbers lie 2^-133 apart
    unit = ((e.long() - 8 + 1023) << 52).view(torch.float64)  # 2^(e - 8), made of its bits: pow need not be exact
    return rounded(x / unit) * unit


def quantise(torch, x):
    """(codes, scale, minimum) of [..., dim]; scale is NaN for vectors with a NaN or an infinity."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    clean = torch.where(bad[..., None], 0.0, x)
    minimum = _eight_bits(torch, clean.amin(-1), torch.floor)
    spread = clean.amax(-1) - minimum
    scale = _eight_bits(torch, spread / 15.0, torch.ceil)
    scale = torch.where(15.0 * scale < spread, scale * (1 + 2.0 ** -7), scale)   # the quotient itself was rounded
    scale = torch.where(spread > 0, scale.clamp(min=2.0 ** -126), 0.0)
    codes = torch.round((clean - minimum[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(0, 15)
    return torch.where(bad[..., None], 0.0, codes).to(torch.uint8), torch.where(bad, math.nan, scale), torch.where(bad, 0.0, minimum)


def append(torch, cache, bs, k, v, slots):
    keep = slots >= 0
    at = slots[keep].long()
    block, off = at // bs, at % bs
    for x, codes_to, params_to in ((k, "k_codes", "k_params"), (v, "v_codes", "v_params")):
        codes, scale, minimum = quantise(torch, x[keep])
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        if codes_to == "k_codes":
            cache[codes_to][block, :, off] = packed
        else:
            shape = cache[codes_to].shape
            pairs = cache[codes_to].view(shape[0], shape[1], bs // 2, shape[3] // 2, 2, 2)
            pairs[block, :, off // 2, :, off % 2] = packed.unflatten(-1, (-1, 2))
        cache[params_to][block, :, off] = torch.stack((scale, minimum), dim=-1).to(torch.bfloat16)
    return cache


def read(torch, cache, bs, slots):
    """((keys, size), (values, size)): 64 bits, [tokens, heads, dim]; size = |minimum| + 15 scale."""
    block, off = slots // bs, slots % bs
    shape = cache["v_codes"].shape
    pairs = cache["v_codes"].view(shape[0], shape[1], bs // 2, shape[3] // 2, 2, 2)
    out = []
    for packed, params in ((cache["k_codes"][block, :, off], cache["k_params"]), (pairs[block, :, off // 2, :, off % 2].flatten(-2), cache["v_params"])):
        codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2).double()
        p = params[block, :, off].double()
        out.append((p[..., 1:] + p[..., :1] * codes, (p[..., 1:].abs() + 15 * p[..., :1]).expand_as(codes)))
    return out


def attention(torch, cache, bs, table, q, lens, new, heads, scale, causal, window, hidden=(), key_rounding=0.0):
    """(out, lse, limit, lse limit) in 64 bits; the limits are those of the kernels' arithmetic, see test_gpu_kv4.py."""
    rows, hq, dim = q.shape
    group = hq // heads
    out, limit = (torch.zeros((rows, hq, dim), dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64, device=q.device)
    lse_limit = torch.zeros_like(lse)
    row = 0
    for r, (total, n) in enumerate(zip(lens, new)):
        if n == 0 or total == 0:
            row += n
            continue
        pos = torch.arange(total, device=q.device)
        slots = table[r, pos // bs].long() * bs + pos % bs
        (k, ks), (v, vs) = read(torch, cache, bs, slots)
        place = total - n + torch.arange(n, device=q.device)[:, None]
        seen = torch.ones((n, total), dtype=torch.bool, device=q.device)
        if causal:
            seen &= pos[None, :] <= place
        if window:
            seen &= pos[None, :] > place - window
        for t in hidden:
            seen[:, t] = False
        some = seen.any(-1)
        for h in range(hq):
            kh, vh = k[:, h // group], v[:, h // group]
            x = q[row:row + n, h].double()
            s = (x @ torch.where(seen.any(0)[:, None], kh, 0.0).T) * scale
            size = (x.abs() @ torch.where(seen.any(0)[:, None], ks[:, h // group], 0.0).nan_to_num(0.0).T) * abs(scale)
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            p = torch.where(seen, torch.exp(s - top), 0.0)
            mass = p.sum(-1, keepdim=True)
            # NaN keys or values spoil the rows that see them and no others
            spoiled = (seen & (kh[:, 0].isnan() | vh[:, 0].isnan())[None, :]).any(-1) | x.isnan().any(-1)
            clean_p = torch.where(spoiled[:, None] | ~some[:, None], 0.0, (p / mass).nan_to_num(0.0))
            clean_v = torch.where(seen.any(0)[:, None], vh, 0.0).nan_to_num(0.0)
            y = clean_p @ clean_v
            score_error = torch.where(seen, size, 0.0).amax(-1) * (2.0 ** -23 * (dim / 16 + 8) + key_rounding)
            weight_error = score_error + 2.0 ** -12 + 2.0 ** -20
            far = torch.where(seen.any(0)[:, None], clean_v, 0.0)
            spread = far.abs().amax() + y.abs().amax(-1, keepdim=True)
            biggest = torch.where(seen.any(0), vs[:, h // group, 0].nan_to_num(0.0), 0.0).amax()
            wide = (clean_p * torch.where(seen.any(0), vs[:, h // group, 0].nan_to_num(0.0), 0.0)[None, :]).sum(-1, keepdim=True)
            limit[row:row + n, h] = 2 * weight_error[:, None] * torch.minimum(spread, 2 * wide) + \
                2.0 ** -23 * (total / 16 + 8) * wide + 2.0 ** -31 * total * biggest
            out[row:row + n, h] = torch.where(spoiled[:, None], math.nan, y)
            value = top[:, 0] + mass[:, 0].log()
            lse[row:row + n, h] = torch.where(spoiled, math.nan, torch.where(some, value, -math.inf))
            lse_limit[row:row + n, h] = score_error + 2.0 ** -22 * (total / 16 + 8) + 2.0 ** -22 * value.abs()
        row += n
    return out, lse, limit, lse_limit
