"""64-bit CPU definitions of the quantised latent cache, the attention over it and the block-scaled 8-bit products
(test infrastructure; plain loops and sums, no code of the package)."""
from __future__ import annotations

import torch

ROW = 656


def e4m3_table() -> torch.Tensor:
    b = torch.arange(256)
    e, f = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * torch.exp2(e.double() - 7))
    v[(b & 127) == 127] = float("nan")
    return torch.where(b >= 128, -v, v)


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    a = v.abs().clamp_max(448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def norm_rotate(kv, gain=None, eps=1e-6, cos=None, sin=None, interleaved=False):
    """(latent [n, 512], position [n, 64]) in 64 bits, before any rounding."""
    x = kv.double()
    n, r = x[:, :512], x[:, 512:576]
    if gain is not None:
        n = n / torch.sqrt((n * n).sum(1, keepdim=True) / 512 + eps) * gain.double()
    if cos is not None:
        c, s, o = cos.double(), sin.double(), torch.empty_like(r)
        for i in range(32):
            u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + 32)
            cu, cv = (i, i) if interleaved else (i, i + 32)
            o[:, u] = r[:, u] * c[:, cu] - r[:, v] * s[:, cu]
            o[:, v] = r[:, v] * c[:, cv] + r[:, u] * s[:, cv]
        r = o
    return n, r


def cache_rows(cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Rows [.., 576] in 64 bits: code * scale, then the position dims."""
    raw = cache.reshape(-1, ROW)[slots]
    codes = e4m3_table()[raw[..., :512].long()]
    scale = raw[..., 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, -1)
    return torch.cat([codes * scale, raw[..., 528:].contiguous().view(torch.bfloat16).double()], -1)


def cache_scales(cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    return cache.reshape(-1, ROW)[slots][..., 512:528].contiguous().view(torch.float32)


def item_keys(idx, table, page, last, base=None, mask=None):
    """Slots of one item's keys in order (selected, then drafted), the ones without a page left out."""
    pos = [int(v) for v in idx if 0 <= int(v) <= last and (base is None or int(v) < base)]
    if mask is not None:
        pos += [base + b for b in range(64) if (int(mask) >> b) & 1]
    return torch.tensor([int(table[v // page]) * page + v % page for v in pos], dtype=torch.long)


def attend(q, rows, scale):
    """ctx [H, 512], lse [H], and sum p |v| [H, 512], max_j sum |q k| [H] for error bounds; q [H, 576], rows [k, 576]."""
    H = q.shape[0]
    if rows.shape[0] == 0:
        z = torch.zeros(H, 512, dtype=torch.float64)
        return z, torch.full((H,), float("-inf"), dtype=torch.float64), z, torch.zeros(H, dtype=torch.float64)
    q = q.double()
    s = q @ rows.t() * scale
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse.view(-1, 1))
    mass = (q.abs() @ rows.abs().t()).amax(1) * scale
    return p @ rows[:, :512], lse, p @ rows[:, :512].abs(), mass


def quantise_groups(x, ue8m0=False, floor=1e-10):
    """(codes as values [M, K], scales [M, G]) in 64 bits."""
    q, sc = torch.empty_like(x, dtype=torch.float64), []
    for k in range(0, x.shape[1], 128):
        g = x[:, k:k + 128].double()
        s = g.abs().amax(1, keepdim=True).clamp_min(floor) / 448.0
        if ue8m0:
            p = torch.exp2(torch.round(torch.log2(s)) - 1)
            while bool((p < s).any()):
                p = torch.where(p < s, 2 * p, p)
            s = p
        q[:, k:k + 128] = round_e4m3(g / s)
        sc.append(s)
    return q, torch.cat(sc, 1)


def block_matmul(a, sa, w, sw):
    """(y, sum of absolute products) in 64 bits; a [M, K], w [N, K] values of the codes."""
    K, N = a.shape[1], w.shape[0]
    x = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    y = w.double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return x @ y.t(), x.abs() @ y.abs().t()
