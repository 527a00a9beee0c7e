"""The cache in 8 bits in plain form: its numbers, its layout, attention in 64 bits, and the stand-in backend with it."""
import math

import torch

from emu_backend import EmuBackend


def quantised(x):
    """(codes, scales) of rows along the last dimension, from the definition in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1).float()
    scale = (top.double() / 127).float().clamp_min(2.0 ** -126)
    bad = ~torch.isfinite(x.float()).all(-1)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    codes = torch.where(bad[..., None], torch.zeros_like(x), (x / scale.double()[..., None]).round())
    return codes.to(torch.int8), scale


def turn(bs, d, device):
    row = torch.arange(bs, device=device)[:, None]
    f = row & 7 if d % 128 == 0 else (row >> 1) & 3 if d % 64 == 0 else row * 0
    return torch.arange(d // 16, device=device)[None, :] ^ f


def pack(k, ks, v, vs):
    """Records from codes [pages, block, G, d] and scales [pages, block, G]."""
    pages, bs, G, d = k.shape
    record = (2 * bs * d + 8 * bs + 15) // 16 * 16
    out = torch.zeros(pages, G, record, dtype=torch.uint8, device=k.device)
    at = turn(bs, d, k.device)[None, None, :, :, None].expand(pages, G, -1, -1, 16)
    for n, (c, s) in enumerate(((k, ks), (v, vs))):
        b = (c.to(torch.int16) + 128).to(torch.uint8).permute(0, 2, 1, 3).reshape(pages, G, bs, d // 16, 16)
        out[..., n * bs * d:(n + 1) * bs * d] = torch.gather(b, 3, at).reshape(pages, G, bs * d)
        out[..., 2 * bs * d + 4 * bs * n:2 * bs * d + 4 * bs * (n + 1)] = s.permute(0, 2, 1).reshape(-1).clone().view(torch.uint8).reshape(pages, G, 4 * bs)
    return out


def unpack(cache, bs, G, d):
    """(key codes, key scales, value codes, value scales) of records."""
    pages, out = cache.shape[0], []
    at = turn(bs, d, cache.device)[None, None, :, :, None].expand(pages, G, -1, -1, 16)
    for n in range(2):
        b = cache[..., n * bs * d:(n + 1) * bs * d].reshape(pages, G, bs, d // 16, 16)
        out.append((torch.gather(b, 3, at).reshape(pages, G, bs, d).permute(0, 2, 1, 3).to(torch.int16) - 128).to(torch.int8))
        s = cache[..., 2 * bs * d + 4 * bs * n:2 * bs * d + 4 * bs * (n + 1)].reshape(-1).clone().view(torch.float32)
        out.append(s.reshape(pages, G, bs).permute(0, 2, 1))
    return out


def values(cache, bs, G, d):
    """Keys and values [pages, block, G, d] in 64 bits."""
    k, ks, v, vs = unpack(cache, bs, G, d)
    return k.double() * ks.double()[..., None], v.double() * vs.double()[..., None]


def rotated(x, table, positions, n_rot, pairing):
    if not n_rot:
        return x
    cs = table[positions.long()][:, None].to(x.dtype)
    c, s, half = cs[..., 0], cs[..., 1], n_rot // 2
    if pairing == "half":
        a, b = x[..., :half], x[..., half:n_rot]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., n_rot:]], -1)
    a, b = x[..., 0:n_rot:2], x[..., 1:n_rot:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), x[..., n_rot:]], -1)


def first_seen(pos, mask):
    return max(0, pos - mask + 1) if mask > 0 else pos // -mask * -mask if mask < 0 else 0


def attention(q, cache, table, token_seq, positions, bs, H, G, d, mask, scale, sinks=None, zero_sink=False, slopes=None, head_scales=None,
              softcap=0.0, missing=()):
    """(outputs [T, H, d], sum of p |v| with the outputs' weights, largest sum of |q| 255 ks scale over the keys, most keys seen times the
    largest value that any scale stands for) in 64 bits.
    ``missing``: (request, block) pairs whose keys are not there."""
    kf, vf = (x.flatten(0, 1) for x in values(cache, bs, G, d))
    T, dev = positions.shape[0], q.device
    qf = q.double().view(T, G, H // G, d)
    out, size = (torch.zeros(T, H, d, dtype=torch.float64, device=dev) for _ in range(2))
    worst = far = 0.0
    _, ks, _, vs = unpack(cache, bs, G, d)
    ksf, vsf = (x.double().flatten(0, 1) for x in (ks, vs))
    for t in range(T):
        pos, s = int(positions[t]), int(token_seq[t])
        key = torch.arange(first_seen(pos, mask), pos + 1, device=dev)
        gone = [b for r, b in missing if r == s]
        if gone:
            key = key[~torch.isin(key // bs, torch.tensor(gone, device=dev))]
        if len(key) == 0 and sinks is None and not zero_sink:
            continue
        at = table[s].long()[key // bs] * bs + key % bs
        a = torch.einsum("grd,kgd->grk", qf[t], kf[at]).reshape(H, -1) * scale
        most = (qf[t].abs().sum(-1)[..., None] * 255 * ksf[at].T[:, None]).max() if len(key) else 0.0
        worst = max(worst, float(most) * scale) if math.isfinite(float(most)) else worst
        if len(key):
            far = max(far, len(key) * 127 * float(vsf[at].nan_to_num(0).max()))
        if head_scales is not None:
            a = a * head_scales.double()[:, None]
        if softcap:
            a = softcap * torch.tanh(a / softcap)
        if slopes is not None:
            a = a - slopes.double()[:, None] * (pos - key)
        if sinks is not None or zero_sink:
            a = torch.cat([a, sinks.double()[:, None] if sinks is not None else torch.zeros(H, 1, dtype=torch.float64, device=dev)], 1)
        p = torch.softmax(a, -1)[:, :len(key)].view(G, H // G, -1)
        out[t] = torch.einsum("grk,kgd->grd", p, vf[at]).reshape(H, d)
        size[t] = torch.einsum("grk,kgd->grd", p, vf[at].abs()).reshape(H, d)
    return out, size, worst, far


class EmuKv8(EmuBackend):
    def kv8_write(self, rows, v, cos_sin, n_rot, pairing, positions, slots, q_out, cache, H, G, d, block_size):
        T = rows.shape[0]
        q, k, v = (None, rows, v) if v is not None else (rows[:, :H * d], rows[:, H * d:(H + G) * d], rows[:, (H + G) * d:])
        if H:
            q_out.copy_(rotated(q.float().reshape(T, H, d), cos_sin, positions, n_rot, pairing).reshape(T, H * d).to(q_out.dtype))
        if slots is None:
            return
        kc, ks, vc, vs = (x.clone() for x in unpack(cache, block_size, G, d))
        ok = slots >= 0
        page, row = slots[ok].long() // block_size, slots[ok].long() % block_size
        kc[page, row], ks[page, row] = quantised(rotated(k.double().reshape(T, G, d), cos_sin, positions, n_rot, pairing)[ok])
        vc[page, row], vs[page, row] = quantised(v.double().reshape(T, G, d)[ok])
        cache.copy_(pack(kc, ks, vc, vs))

    def kv8_read(self, cache, pages, rows, k_out, v_out, N, bs, G, d):
        used = (torch.arange(bs, device=cache.device)[None] < rows[:, None]) & (pages >= 0)[:, None]
        for out, x in zip((k_out, v_out), values(cache, bs, G, d)):
            out.copy_(torch.where(used[..., None, None], x[pages.long().clamp_min(0)], torch.zeros((), dtype=torch.float64, device=cache.device)))

    def paged_attention_kv8(self, q, cache, meta, ctx, H, G, d, window, scale, out, tiles, settled=False, **options):
        T = q.shape[0]
        o = attention(q, cache, meta.block_table, ctx.token_seq[:T], ctx.positions[:T], meta.block_size, H, G, d, window, scale, **options)[0]
        out.copy_(o.reshape(T, H * d).to(out.dtype))
