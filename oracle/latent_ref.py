"""Latent cache and latent attention in 64-bit torch, from their definitions (test infrastructure).

A row of the cache holds a latent c in 4 bits and a rotary key in fp16: per 64 values y = H c with the
normalised Sylvester Hadamard matrix H, s = clamp(bf16(max|y| * fp32(1/7)), 2^-14, 2048) and
n = clamp(rint(y / s), -7, 7); it stands for H (n s)."""
import math

import torch


def hadamard(n=64):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < n:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / math.sqrt(n)


def row_bytes(L, R):
    return (L // 2 + 2 * R + 2 * (L // 64) + 15) // 16 * 16


def quantise(c):
    """c [N, L] -> (n int64 [N, L], s fp64 [N, L/64])."""
    N, L = c.shape
    y = c.double().reshape(N, L // 64, 64) @ hadamard().to(c.device)
    m = y.abs().amax(-1).float() * torch.tensor(1.0 / 7.0, dtype=torch.float32, device=c.device)
    s = m.bfloat16().double().clamp(2.0 ** -14, 2048.0)
    return torch.round(y / s[..., None]).clamp(-7, 7).long().reshape(N, L), s


def pack_rows(c, k_rope):
    """The cache rows, u8 [N, row_bytes]."""
    n, s = quantise(c)
    N, L = c.shape
    w = torch.zeros(N, L // 8, dtype=torch.int64, device=c.device)
    for j in range(8):
        w |= (n.reshape(N, L // 8, 8)[..., j] + 8) << (4 * (j >> 1) + 16 * (j & 1))
    parts = [torch.stack([(w >> (8 * k)) & 255 for k in range(4)], -1).reshape(N, L // 2).to(torch.uint8),
             k_rope.double().clamp(-65504, 65504).half().contiguous().view(torch.uint8).reshape(N, -1),
             s.half().view(torch.uint8).reshape(N, -1)]
    rows = torch.cat(parts, 1)
    return torch.cat((rows, rows.new_zeros(N, row_bytes(L, k_rope.shape[1]) - rows.shape[1])), 1)


def unpack_rows(rows, L, R):
    """(c', k_rope') in fp64 of cache rows u8 [N, row_bytes]."""
    N = rows.shape[0]
    w = rows[:, : L // 2].long().reshape(N, L // 8, 4)
    w = w[..., 0] | (w[..., 1] << 8) | (w[..., 2] << 16) | (w[..., 3] << 24)
    n = torch.stack([((w >> (4 * (j >> 1) + 16 * (j & 1))) & 15) - 8 for j in range(8)], -1).double()
    s = rows[:, L // 2 + 2 * R: L // 2 + 2 * R + L // 32].contiguous().view(torch.float16).double()
    y = n.reshape(N, L // 64, 64) * s[..., None]
    kr = rows[:, L // 2: L // 2 + 2 * R].contiguous().view(torch.float16).double()
    return (y @ hadamard().to(rows.device)).reshape(N, L), kr.reshape(N, R)


def attend(q, k, v, last, scale):
    """q [n, D], k [m, D], v [m, dv]; row i sees keys j <= last[i]. Returns (out, sum_j p_j |v_j|)."""
    n, m = q.shape[0], k.shape[0]
    out = torch.zeros(n, v.shape[1], dtype=torch.float64, device=q.device)
    absolute = torch.zeros_like(out)
    if m == 0:
        return out, absolute
    z = (q.double() @ k.double().T) * scale
    z = z.masked_fill(torch.arange(m, device=q.device)[None, :] > last[:, None], -math.inf)
    p = torch.softmax(z, -1)
    p = torch.where((last < 0)[:, None], 0.0, p)
    return p @ v.double(), p @ v.double().abs()


def decode(q, data, table, kv_len, scale, L, R):
    """q [B, T, heads, L + R] over cache data u8 [pages, page_size, row_bytes]."""
    B, T, heads, D = q.shape
    page = data.shape[1]
    flat = data.reshape(-1, data.shape[2])
    out = torch.zeros(B, T, heads, L, dtype=torch.float64, device=q.device)
    absolute = torch.zeros_like(out)
    for b in range(B):
        n = int(kv_len[b])
        if n <= 0:
            continue
        at = torch.arange(n, device=q.device)
        c, kr = unpack_rows(flat[table[b, at // page].long() * page + at % page], L, R)
        last = (n - T + torch.arange(T, device=q.device)).repeat_interleave(heads)
        o, a = attend(q[b].reshape(T * heads, D), torch.cat((c, kr), 1), c, last, scale)
        out[b], absolute[b] = o.reshape(T, heads, L), a.reshape(T, heads, L)
    return out, absolute


def prefill(q, k_nope, k_rope, v, cu_q, cu_k, scale):
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
    absolute = torch.zeros_like(out)
    for b in range(len(cu_q) - 1):
        (i, j), (x, y) = (int(cu_q[b]), int(cu_q[b + 1])), (int(cu_k[b]), int(cu_k[b + 1]))
        last = torch.arange(j - i, device=q.device) + (y - x) - (j - i)
        for h in range(q.shape[1]):
            k = k_nope[x:y, h].double()
            if k_rope is not None:
                k = torch.cat((k, k_rope[x:y].double()), 1)
            out[i:j, h], absolute[i:j, h] = attend(q[i:j, h], k, v[x:y, h], last, scale)
    return out, absolute
