"""Plain 64-bit forms of the 8-bit blocks, their product and the RMS norm (test infrastructure)."""
import torch

BLOCK = 128


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Doubles of at most 448 (1 + 2^-20) in magnitude to the nearest e4m3 value, ties to even."""
    part, _ = torch.frexp(v)
    step = torch.where(v == 0, torch.ones_like(v), v / part / 16).clamp(min=2.0**-9)
    return (torch.round(v / step) * step).clamp(-448, 448)


def f32(v: torch.Tensor) -> torch.Tensor:
    return v.to(torch.float32).double()


def scales_of(x: torch.Tensor, square: bool = False) -> torch.Tensor:
    """Of a matrix of doubles: [rows, blocks], or [blocks of rows, blocks]."""
    m, k = x.shape
    pad = torch.nn.functional.pad(x.abs(), (0, -k % BLOCK, 0, -m % BLOCK if square else 0))
    top = pad.view(-1, BLOCK if square else 1, pad.shape[1] // BLOCK, BLOCK).amax((1, 3))
    return f32(top / 448).clamp(min=2.0**-126)


def spread(s: torch.Tensor, shape, square: bool) -> torch.Tensor:
    """A scale per element."""
    if square:
        s = s.repeat_interleave(BLOCK, 0)[:shape[0]]
    return s.repeat_interleave(BLOCK, 1)[:, :shape[1]]


def quantize(x: torch.Tensor, square: bool = False):
    """(values, scales) as doubles on the CPU; x of any type."""
    x = x.detach().cpu().double()
    s = scales_of(x, square)
    return round_e4m3(f32(x * spread(f32(1 / s), x.shape, square))), s


def held(x: torch.Tensor, square: bool = False) -> torch.Tensor:
    """What the 8-bit form of x stands for."""
    q, s = quantize(x, square)
    return q * spread(s, q.shape, square)


def held_by(t) -> torch.Tensor:
    """What an Fp8Tensor stands for, as a matrix of doubles on the CPU."""
    k = t.shape[-1]
    q = t.values.reshape(-1, k).cpu().float().double()
    s = t.scales.cpu().double()
    return q * spread(s if t.square else s.reshape(-1, s.shape[-1]), q.shape, t.square)


def product_bound(a: torch.Tensor, b: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What the sums of a b^T may be off by before they are rounded to `dtype`.

    fp32: within a block of 128 at most 128 additions, each off by at most a step (2^-23, an addition that cuts counts) of a partial sum,
    which is at most sum |a b|: 2^-16 of it; then a multiplication by each of two scales, whose own product is rounded, and an addition
    per block, half a step of at most the sum each.
    16 bits: the matrix cores' 8-bit products of 8 neighbouring k are cut at 2^-13 of the largest one's power of two, so that each of the
    other 7 loses at most 2^-13 of that product."""
    blocks = -(-a.shape[1] // BLOCK)
    bound = (2.0**-16 + (blocks + 3) * 2.0**-24) * (a.abs() @ b.abs().t())
    if dtype == torch.float32:
        return bound
    at = "cuda" if torch.cuda.is_available() else "cpu"
    largest = torch.zeros(bound.shape, device=at)
    x, y = a.abs().float().to(at), b.abs().float().to(at)
    for g in range(0, a.shape[1], 8):
        m = torch.zeros_like(largest)
        for k in range(g, min(g + 8, a.shape[1])):
            m = torch.maximum(m, x[:, k, None] * y[None, :, k])
        largest += m
    return bound + 7 * 2.0**-13 * largest.cpu().double()
