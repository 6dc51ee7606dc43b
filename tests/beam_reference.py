"""A beam search's step and the words' embeddings from their definitions, in 64 bits on the CPU: what the
kernels are held to."""
import numpy as np
import torch

import node_reference as nodes


def extend(E, P, frames, positions, scores, width):
    """scores float64, parents, words [B, width]."""
    z, here = nodes.scores(E, P, frames, positions)
    scores = scores.detach().cpu()
    B, N, V = z.shape
    d = torch.full((B, N, V + 1), -torch.inf, dtype=torch.float64)
    bad = torch.zeros(B, dtype=torch.bool)
    for b in range(B):
        for n in range(N):
            s = scores[b, n]
            if s == -torch.inf:
                continue
            if not s < torch.inf:
                bad[b] = True
            elif not here[b, n]:
                d[b, n, 0] = s
            else:
                x = z[b, n].double()
                if not (x < torch.inf).all():
                    bad[b] = True
                elif (x > -torch.inf).any():
                    x -= x.max()   # (exact, or next to it: also where masked words are as low as their type goes)
                    d[b, n, 1:] = s.double() + (x - x.exp().sum().log())
    d = d.flatten(1)
    if d.shape[1] < width:
        d = torch.nn.functional.pad(d, (0, width - d.shape[1]), value=-torch.inf)
    d, at = torch.sort(d, dim=1, descending=True, stable=True)
    d, at = d[:, :width].clone(), at[:, :width]
    left = (d == -torch.inf) | bad[:, None]
    parents = (at // (V + 1)).masked_fill(left, -1)
    words = (at % (V + 1) - 1).masked_fill(left, -1)
    d[bad] = torch.nan
    return d, parents.int(), words.int()


def philox(counter, key):
    """Philox4x32-10: counter [..., 4] and key (2 numbers) to [..., 4], uint64 arrays of 32-bit numbers."""
    low = np.uint64(0xffffffff)
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [np.uint64(x) for x in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xd2511f53), c[2] * np.uint64(0xcd9e8d57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9e3779b9)) & low, (k[1] + np.uint64(0xbb67ae85)) & low]
    return np.stack(c, -1)


def kept(count, H, dropout, seed):
    """bool [count, H]: the numbers that stay."""
    k = min(65535, round(dropout * 65536))
    groups = (H + 7) // 8
    counter = np.zeros((count, groups, 4), np.uint64)
    counter[..., 0] = np.arange(count)[:, None]
    counter[..., 2] = np.arange(groups)
    seed = seed % 2 ** 64
    x = philox(counter, (seed % 2 ** 32, seed // 2 ** 32))
    halves = np.stack((x & np.uint64(0xffff), x >> np.uint64(16)), -1).reshape(count, groups * 8)
    return torch.from_numpy(halves[:, :H] >= k)


def factor(scale, dropout):
    k = min(65535, round(dropout * 65536))
    return scale * 65536 / (65536 - k)


def embed(table, words, scale=1.0, dropout=0.0, seed=0):
    """rows float64 [words, H], and which numbers count."""
    table, words = table.detach().cpu().double(), words.cpu().flatten().long()
    R, H = table.shape
    here = ((words >= 0) & (words < R))[:, None].expand(-1, H)
    if dropout > 0.0:
        here = here & kept(words.numel(), H, dropout, seed)
    at = words.clamp(min=0, max=max(R - 1, 0))
    rows = table[at] if R else torch.zeros(words.numel(), H, dtype=torch.float64)
    return torch.where(here, rows * factor(scale, dropout), 0.0), here


def embed_grad(R, words, deltas, here, scale=1.0, dropout=0.0):
    """grad float64 [R, H], the sum of the summands' magnitudes, and their greatest number."""
    words, deltas = words.cpu().flatten().long(), deltas.detach().cpu().double().flatten(0, -2)
    f = factor(scale, dropout)
    x = torch.where(here, deltas * f, 0.0)
    at = words.clamp(min=0, max=max(R - 1, 0))
    valid = (words >= 0) & (words < R)
    x, at = x[valid], at[valid]
    grad = torch.zeros(R, deltas.shape[-1], dtype=torch.float64).index_add_(0, at, x)
    size = torch.zeros_like(grad).index_add_(0, at, x.abs())
    return grad, size, torch.bincount(at, minlength=R)[:, None].double()
