"""Plain 64-bit forms of residual dropout, its sum with LayerNorm, and the relative position bias (test infrastructure)."""
import numpy as np
import torch

M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key, rounds=10):
    """Philox4x32 of Salmon, Moraes, Dror and Shaw (2011): counter [..., 4] and key (2) of 32-bit numbers -> [..., 4]."""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & M32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & M32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def keep_mask(shape, p, seed, shared_dim=None) -> torch.Tensor:
    """Truth values of `shape` (CPU): which elements stay."""
    sizes = list(shape)
    if shared_dim is not None:
        sizes[shared_dim] = 1
    cols, rows = sizes[-1], int(np.prod(sizes[:-1]))
    blocks = -(-cols // 8)
    counter = np.zeros((rows, blocks, 4), np.uint64)
    counter[..., 0] = np.arange(blocks)[None, :]
    counter[..., 1] = np.arange(rows)[:, None]
    u = np.zeros((rows, blocks, 8), np.uint64)
    for draw in (0, 1):
        counter[..., 3] = draw
        w = philox(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
        halves = np.stack((w & np.uint64(0xFFFF), w >> np.uint64(16)), -1).reshape(rows, blocks, 8)
        u = (u << np.uint64(16)) | halves
    keep = (u.reshape(rows, blocks * 8)[:, :cols] >= np.uint64(round(p * 2.0**32))).reshape(sizes)
    return torch.from_numpy(keep.copy()).expand(shape).contiguous()


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def smallest(dtype: torch.dtype) -> float:
    """Half the smallest subnormal: what a rounding is off by near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def update(x, residual, p, seed, shared_dim):
    """(h, m) in 64 bits on the CPU: the sum and the factor of every element of x (0 where dropped)."""
    x = x.detach().cpu().double()
    m = torch.ones_like(x)
    if p > 0:
        m = keep_mask(x.shape, p, seed, shared_dim).double() * (1.0 / (1.0 - p) if p < 1 else 0.0)
    kept = torch.where(m != 0, x * m, torch.zeros_like(x))
    return kept if residual is None else residual.detach().cpu().double() + kept, m


def norm_parts(h, weight, bias, eps):
    """y, xh and rstd of the LayerNorm of h, in 64 bits."""
    mean = h.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((h - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (h - mean) * rstd
    w = 1.0 if weight is None else weight.detach().cpu().double()
    b = 0.0 if bias is None else bias.detach().cpu().double()
    return xh * w + b, xh, rstd


def bucket(d, max_distance, num_buckets=None, bidirectional=True):
    """The bucket of a whole-number difference key - query, from the formula in whole numbers."""
    if num_buckets is None:
        return max_distance + max(-max_distance, min(max_distance, d)) if bidirectional else min(max(-d, 0), max_distance)
    side = num_buckets // 2 if bidirectional else num_buckets
    n = abs(d) if bidirectional else max(-d, 0)
    upper = side if bidirectional and d > 0 else 0
    e = side // 2
    if n < e:
        return upper + n
    s, j = side - e, 0
    while j + 1 < s and n**s >= max_distance ** (j + 1) * e ** (s - j - 1):
        j += 1
    return upper + e + j
