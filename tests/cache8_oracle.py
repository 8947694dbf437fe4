"""The 8-bit cache and the row rotation in plain form, on the CPU: what the
GPU tests compare with."""

import numpy as np
import torch

CODE = torch.float8_e4m3fn
ROW_EPS = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative


def scale_for(amax):
    """The smallest power of two >= amax / 448, at least 2^-64 (a loop: the
    definition itself)."""
    e = -64
    while 448.0 * 2.0**e < amax:
        e += 1
    return 2.0**e


def write(codes, scales, rows, slots):
    """Append ``rows`` [T, H, D] (fp32, the values the 16-bit cache would hold)
    to ``codes`` [N, bs, H, D] / ``scales`` [N, H], both modified."""
    blocks, bs, heads, dim = codes.shape
    groups = {}
    for t, slot in enumerate(slots):
        if 0 <= slot < blocks * bs:
            groups.setdefault(slot // bs, []).append(t)
    for block, tokens in groups.items():
        at = [slots[t] % bs for t in tokens]
        for h in range(heads):
            x = rows[tokens, h]
            finite = x[torch.isfinite(x)].abs()
            scale = scale_for(float(finite.max()) if finite.numel() else 0.0)
            if 0 not in at:
                old = float(scales[block, h])
                scale = max(scale, old)
                if scale != old:
                    codes[block, :, h] = (codes[block, :, h].float() * (old / scale)).to(CODE)
            code = (x / scale).to(CODE)
            code.view(torch.uint8)[~torch.isfinite(x)] = torch.where(torch.signbit(x[~torch.isfinite(x)]), 0xFF,
                                                                     0x7F).to(torch.uint8)
            codes[block, at, h] = code
            scales[block, h] = scale
    return codes, scales


def values(codes, scales):
    """[N, bs, H, D] in fp64."""
    return codes.float().double() * scales.double()[:, None, :, None]


def rotated(x, weight, positions, cos_sin, eps, interleaved):
    """Rows [T, H, D] normalised and rotated in fp64, and the magnitude its
    rounding errors scale with (|a| + |b| of each pair, normalised)."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    r = cos_sin.shape[1]
    cs = cos_sin.double()[positions][:, None]
    c, s = cs[..., : r // 2], cs[..., r // 2 :]
    i = torch.arange(r // 2)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    out, size = x.clone(), x.abs()
    out[..., one] = x[..., one] * c - x[..., two] * s
    out[..., two] = x[..., two] * c + x[..., one] * s
    size[..., one] = size[..., two] = x[..., one].abs() + x[..., two].abs()
    return out, size


def attention(q, keys, vals, table, starts, counts, scale):
    """Causal attention of each sequence's new tokens over its blocks in fp64:
    the result, the weighted mean of |v| beside it, and the largest weight times
    the sum of |v|.  Positions whose block is missing are skipped; a row that
    attends nothing is zero."""
    total, bs, hkv, dim = keys.shape
    group = q.shape[1] // hkv
    out, size, peak = [], [], []
    at = 0
    for row, start, count in zip(table, starts, counts):
        end = start + count
        pos = np.arange(end)
        col = pos // bs
        blk = np.where(col < len(row), np.asarray(row)[np.minimum(col, len(row) - 1)], -1) if len(row) else -np.ones(end)
        ok = (blk >= 0) & (blk < total)
        slots = torch.from_numpy((blk * bs + pos % bs)[ok].astype(np.int64))
        k = keys.reshape(-1, hkv, dim)[slots].repeat_interleave(group, 1).transpose(0, 1)  # [H, n, D]
        v = vals.reshape(-1, hkv, dim)[slots].repeat_interleave(group, 1).transpose(0, 1)
        p = torch.from_numpy(pos[ok])
        later = p[None, :] > start + torch.arange(count)[:, None]
        w = torch.matmul(q[at:at + count].double().transpose(0, 1), k.transpose(1, 2)) * scale
        w = torch.nan_to_num(torch.softmax(w.masked_fill(later, -float("inf")), dim=-1)) if p.numel() else w
        out.append(torch.matmul(w, v).transpose(0, 1))
        size.append(torch.matmul(w, v.abs()).transpose(0, 1))
        most = w.amax(-1, keepdim=True) if p.numel() else w.sum(-1, keepdim=True)
        peak.append(torch.matmul((w > 0).double() * most, v.abs()).transpose(0, 1))
        at += count
    return torch.cat(out), torch.cat(size), torch.cat(peak)
