"""What a block's residual updates and its attention bias take in training and in serving, beside the
attention operator and LayerNorm: the calls, their plain forms and their definitions in 64 bits.

    dropout_add              residual + dropout(x): the mask comes from a counter-based generator and is never stored
    dropout_add_layer_norm   the same sum and the LayerNorm of it that the next update reads (p = 0: serving)
    relative_position_bias   a learned bias per head and bucket of relative position, the attention operator's Bias2

Each case is a dict of plain values.  `mode` names the storage types as "<x>" or "<x>/<residual>"; a pass is forward
and backward where `backward` is true (the gradients belong to its outputs), else forward only.

The dropout mask (Philox4x32-10; Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011): with
the rows of the mask numbered r and columns in blocks of 8, block k of row r takes its eight 16-bit halves
from the counter (k, r mod 2^32, r div 2^32, 0) under the seed as key, low half first; the same halves of the counter (k, ., ., 1) are
the lower 16 bits of a 32-bit number u, and an element is kept where u >= round(p 2^32).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_MODES = ["fp32", "bf16", "fp16", "bf16/fp32", "fp16/fp32"]


def _add(shape, mode, p, shared_dim=None, residual=True):
    return {"op": "dropout_add", "shape": "x".join(map(str, shape)), "mode": mode, "p": p, "shared_dim": shared_dim or 0,
            "residual": residual, "backward": True}


def _norm(shape, mode, p, shared_dim=None, residual=True, backward=True, weights="fp32"):
    return {"op": "dropout_add_layer_norm", "shape": "x".join(map(str, shape)), "mode": mode, "p": p,
            "shared_dim": shared_dim or 0, "residual": residual, "backward": backward, "weights": weights}


def _bias(batch, heads, q, k, mode, max_distance, num_buckets=0, bidirectional=True, positions="range", backward=True):
    # num_buckets 0: one bucket per distance up to max_distance; positions "range": keys 0 .. k - 1, queries the last
    # q of them; "chains": residue numbers that start again in every chain, chains apart in a bucket of their own
    return {"op": "relative_position_bias", "batch": batch, "heads": heads, "q": q, "k": k, "mode": mode,
            "max_distance": max_distance, "num_buckets": num_buckets, "bidirectional": bidirectional,
            "positions": positions, "backward": backward}


def listed():
    return [
        # the single track of a small complex: a few microseconds of memory traffic, launches and the host count
        dict(_add((1, 93, 384), "bf16", 0.1), name="dropout_add_single_n93"),
        # rows of a length that nothing divides, a mask shared along the columns
        dict(_add((2, 147, 211, 67), "fp16", 0.15, shared_dim=-2), name="dropout_add_odd_columns"),
        # a batch of sequences, every element with a draw of its own
        dict(_add((8, 1024, 768), "bf16", 0.1), name="dropout_add_sequences"),
        # the update of the pair tensor at the benchmark's 768 tokens, in bf16 onto the fp32 residual stream, one
        # mask for all rows of a column as the pair stack's dropout has it
        dict(_add((1, 768, 768, 128), "bf16/fp32", 0.25, shared_dim=-3), name="dropout_add_pair_n768"),
        # serving: the residual sum and the norm in front of the next layer for one token
        dict(_norm((1, 1, 384), "bf16", 0.0, backward=False, weights="bf16"), name="add_norm_one_token"),
        # odd rows and columns in full precision
        dict(_norm((5, 411, 1035), "fp32", 0.1), name="dropout_add_norm_odd"),
        # training on a crop of 384 tokens: an update of the pair tensor and the norm of the next one
        dict(_norm((1, 384, 384, 128), "bf16/fp32", 0.25, shared_dim=-3), name="dropout_add_norm_pair_n384"),
        # training on long sequences of wide rows
        dict(_norm((4, 4096, 2048), "bf16", 0.1), name="dropout_add_norm_wide"),
        # serving: one query behind a long context
        dict(_bias(1, 16, 1, 4001, "bf16", 128, 32, bidirectional=False, backward=False), name="position_bias_one_query"),
        # the pair stack's triangle bias at the benchmark's size, distances to 32 one by one as residues are encoded
        dict(_bias(1, 4, 768, 768, "bf16", 32), name="position_bias_n768"),
        # a batch of crops through several chains each, the single track's 16 heads, in full precision
        dict(_bias(3, 16, 411, 411, "fp32", 32, positions="chains"), name="position_bias_chains"),
        # long sequences, buckets that widen with the distance
        dict(_bias(2, 16, 2048, 2048, "bf16", 128, 32), name="position_bias_long"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dropout_add", "dropout_add_layer_norm", "relative_position_bias"])
    if op == "relative_position_bias":
        heads = rng.choice([1, 3, 4, 8, 16])
        batch = rng.choice([1, 1, 2, 5])
        k = _log_int(rng, 1, 4096)
        q = 1 if rng.random() < 0.25 else _log_int(rng, 1, k)
        q = max(1, min(q, (1 << 26) // (heads * batch * k)))
        linear = rng.random() < 0.5
        both = rng.random() < 0.6
        if linear:
            distance, buckets = rng.choice([1, 8, 32, rng.randint(2, 120)]), 0
        else:
            buckets = 2 * rng.randint(4, 64)
            distance = _log_int(rng, buckets, 4096)
        return _bias(batch, heads, q, k, rng.choice(list(_TYPES)), distance, buckets, both,
                     rng.choice(["range", "chains"]), rng.random() < 0.7)
    p = rng.choice([0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    mode = rng.choice(_MODES)
    if op == "dropout_add":
        cols = rng.choice([64, 128, 384, 768, 1024, 4096, _log_int(rng, 1, 2000), _log_int(rng, 1, 2000)])
        room = (1 << 26) // cols
        a = _log_int(rng, 1, max(1, min(1024, room // 4)))
        b = _log_int(rng, 1, max(1, min(4096, room // a)))
        lead = rng.choice([1, 1, 2, 3]) if a * b * 3 <= room else 1
        return _add((lead, a, b, cols), mode, p, rng.choice([None, None, -2, -3]), rng.random() < 0.85)
    cols = rng.choice([64, 128, 256, 384, 768, 1024, 4096, _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)])
    room = (1 << 25) // cols
    a = _log_int(rng, 1, max(1, min(512, room // 4)))
    b = _log_int(rng, 1, max(1, room // a))
    serving = rng.random() < 0.25
    return _norm((1, a, b, cols), mode, 0.0 if serving else p, None if serving else rng.choice([None, None, -2, -3]),
                 rng.random() < 0.85, not serving, rng.choice(["fp32", mode.split("/")[0]]))


def _shape(case):
    return tuple(int(n) for n in case["shape"].split("x"))


def _types(case):
    x, _, residual = case["mode"].partition("/")
    return _TYPES[x], _TYPES[residual or x]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0, shift=0.0, grad=False):
        t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(dtype).requires_grad_(grad)

    grad = case["backward"]
    if case["op"] == "relative_position_bias":
        return _prepare_bias(case, seed, gen, normal)
    shape = _shape(case)
    tx, tr = _types(case)
    out_type = tr if case["residual"] else tx
    st = {"case": case, "p": case["p"], "shared_dim": case["shared_dim"] or None,
          # the step's seed, a whole number of 64 bits
          "seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63),
          # an update, and the residual stream it is added to, which has grown over the blocks
          "x": normal(shape, tx, 0.7, grad=grad),
          "residual": normal(shape, tr, 3.0, 0.4, grad=grad) if case["residual"] else None}
    if case["op"] == "dropout_add":
        st["dout"] = normal(shape, out_type)
        return st
    tw = _TYPES[case["weights"]]
    st["weight"] = normal(shape[-1:], tw, 0.1, 1.0, grad=grad)
    st["bias"] = normal(shape[-1:], tw, 0.1, grad=grad)
    if grad:
        st["dy"], st["dh"] = normal(shape, tx), normal(shape, out_type)
    return st


def _prepare_bias(case, seed, gen, normal):
    B, H, q, k = (case[n] for n in ("batch", "heads", "q", "k"))
    chains = case["positions"] == "chains"
    dtype = _TYPES[case["mode"]]
    rows = _bucket_count(case) + int(chains)
    st = {"case": case, "table": normal((rows, H), torch.float32, 0.5, grad=case["backward"]), "dtype": dtype, "groups": None}
    if chains:
        # residue numbers of chains of some 30 to 300, some of them starting elsewhere than at 1
        rng = np.random.default_rng(seed)
        pos, grp = np.zeros((B, k), np.int64), np.zeros((B, k), np.int64)
        for b in range(B):
            at, chain = 0, 0
            while at < k:
                n = min(int(rng.integers(30, 300)), k - at)
                pos[b, at:at + n] = int(rng.integers(-4, 40)) + np.arange(n)
                grp[b, at:at + n] = chain
                at, chain = at + n, chain + 1
        kp, kg = torch.from_numpy(pos).cuda(), torch.from_numpy(grp).cuda()
        st["k_pos"], st["q_pos"] = kp, kp[:, k - q:].contiguous()
        st["groups"] = (kg[:, k - q:].contiguous(), kg)
    else:
        st["k_pos"], st["q_pos"] = range(k), range(k - q, k)
    if case["backward"]:
        # the attention's gradient for its bias: rows of a softmax, small almost everywhere
        st["dout"] = normal((B, H, q, k) if chains or B > 1 else (H, q, k), dtype, 0.05)
    if B > 1 and not chains:
        st["q_pos"] = torch.arange(k - q, k, device="cuda").expand(B, q).contiguous()
        st["k_pos"] = torch.arange(k, device="cuda").expand(B, k).contiguous()
    if own:
        import protenix_amd as P

        st["buckets"] = P.RelativeBuckets(case["max_distance"], case["num_buckets"] or None, bidirectional=case["bidirectional"])
    return st


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


# ---- the framework's calls -------------------------------------------------------------------------
def _wanted(*tensors):
    return [t for t in tensors if t is not None]


def _own_add(st):
    import protenix_amd as P

    out = P.dropout_add(st["x"], st["residual"], st["p"], shared_dim=st["shared_dim"], seed=st["seed"])
    return (out, *torch.autograd.grad(out, _wanted(st["x"], st["residual"]), st["dout"]))


def _own_norm(st):
    import protenix_amd as P

    y, h = P.dropout_add_layer_norm(st["x"], st["residual"], st["weight"], st["bias"], st["p"], shared_dim=st["shared_dim"],
                                    seed=st["seed"])
    if not st["case"]["backward"]:
        return y, h
    return (y, h, *torch.autograd.grad((y, h), _wanted(st["x"], st["residual"], st["weight"], st["bias"]), (st["dy"], st["dh"])))


def _own_bias(st):
    import protenix_amd as P

    out = P.relative_position_bias(st["table"], st["buckets"], st["q_pos"], st["k_pos"], groups=st["groups"], dtype=st["dtype"])
    if not st["case"]["backward"]:
        return out
    return (out, *torch.autograd.grad(out, [st["table"]], st["dout"]))


_run_own = {"dropout_add": _own_add, "dropout_add_layer_norm": _own_norm, "relative_position_bias": _own_bias}


# ---- the plain forms -------------------------------------------------------------------------------
_M32 = 0xFFFFFFFF


def _philox(c0, c1, c2, draw, seed):
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    c3 = torch.full_like(c0, draw)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _M32) ^ c1 ^ k0, b & _M32, ((a >> 32) & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), -1)


def _keep(shape, p, shared_dim, seed):
    """The elements that stay, with size 1 along the shared dimension."""
    mask = list(shape)
    if shared_dim:
        mask[shared_dim] = 1
    cols = mask[-1]
    rows = math.prod(mask[:-1])
    blocks = (cols + 7) // 8
    r = torch.arange(rows, device="cuda")[:, None].expand(rows, blocks)
    c = torch.arange(blocks, device="cuda")[None, :].expand(rows, blocks)
    halves = []
    for d in range(2):
        w = _philox(c, r & _M32, r >> 32, d, seed)
        halves.append(torch.stack((w & 0xFFFF, w >> 16), -1).reshape(rows, blocks * 8)[:, :cols])
    u = halves[0] * 65536 + halves[1]
    return (u >= round(p * 2.0**32)).reshape(mask)


def _plain_sum(st):
    """(the sum, which elements stay or None, the factor of those), in 32 bits."""
    x = st["x"].detach().float()
    keep, scale = None, 1.0
    if st["p"] > 0:
        keep, scale = _keep(x.shape, st["p"], st["shared_dim"], st["seed"]), 1.0 / (1.0 - st["p"])
        x = torch.where(keep, x * scale, torch.zeros_like(x))
    return (x if st["residual"] is None else st["residual"].detach().float() + x), keep, scale


def _plain_dx(st, g, keep, scale):
    return (g if keep is None else torch.where(keep, g * scale, torch.zeros_like(g))).to(st["x"].dtype)


def _plain_add(st):
    h, keep, scale = _plain_sum(st)
    res = st["residual"]
    out = [h.to(st["dout"].dtype), _plain_dx(st, st["dout"].float(), keep, scale)]
    return tuple(out if res is None else out + [st["dout"]])


def _plain_norm(st):
    h, keep, scale = _plain_sum(st)
    x, res, w, b = st["x"], st["residual"], st["weight"].detach().float(), st["bias"].detach().float()
    xc = h - h.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xc = xc * rstd
    h_type = x.dtype if res is None else res.dtype
    out = [(xc * w + b).to(x.dtype), h.to(h_type)]
    if not st["case"]["backward"]:
        return tuple(out)
    dy = st["dy"].float()
    g = dy * w
    dh = rstd * (g - g.mean(-1, keepdim=True) - xc * (g * xc).mean(-1, keepdim=True)) + st["dh"].float()
    out.append(_plain_dx(st, dh, keep, scale))
    if res is not None:
        out.append(dh.to(res.dtype))
    dims = tuple(range(dy.dim() - 1))
    tw = st["weight"].dtype
    return (*out, (dy * xc).sum(dims, dtype=torch.float64).to(tw), dy.sum(dims, dtype=torch.float64).to(tw))


def _sides(case):
    """(buckets of one direction, how many of them stand for one distance each)."""
    if not case["num_buckets"]:
        return case["max_distance"] + 1, case["max_distance"] + 1
    side = case["num_buckets"] // 2 if case["bidirectional"] else case["num_buckets"]
    return side, side // 2


def _bucket_count(case):
    return case["num_buckets"] or (2 * case["max_distance"] + 1 if case["bidirectional"] else case["max_distance"] + 1)


def _steps(case):
    """The distances at which the next of the widening buckets begins: bucket e + j, e the number of exact ones, holds
    the distances n with (n / e)^s >= (M / e)^j, s the number of widening ones, in whole numbers."""
    side, e = _sides(case)
    s, top = side - e, case["max_distance"]
    steps = []
    for j in range(1, s):
        bound = top**j * e ** (s - j)
        lo, hi = e, top
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid**s >= bound else (mid + 1, hi)
        steps.append(lo)
    return steps


def _positions(st):
    def tensor(p):
        return torch.arange(p.start, p.stop, device="cuda") if isinstance(p, range) else p

    return tensor(st["q_pos"]), tensor(st["k_pos"])


def _plain_buckets(st):
    case = st["case"]
    q, k = _positions(st)
    d = k[..., None, :] - q[..., :, None]
    top, both = case["max_distance"], case["bidirectional"]
    if not case["num_buckets"]:
        bucket = d.clamp(-top, top) + top if both else (-d).clamp(0, top)
    else:
        side, e = _sides(case)
        n = d.abs() if both else (-d).clamp(min=0)
        bucket = n.clamp(max=e)
        for step in _steps(case):
            bucket = bucket + (n >= step)
        if both:
            bucket = bucket + side * (d > 0)
    if st["groups"] is not None:
        gq, gk = st["groups"]
        bucket = torch.where(gk[..., None, :] == gq[..., :, None], bucket, torch.full_like(bucket, _bucket_count(case)))
    return bucket


def _plain_bias(st):
    bucket = _plain_buckets(st)
    table = st["table"].detach().to(st["dtype"])
    out = table[bucket].movedim(-1, -3).contiguous()
    if not st["case"]["backward"]:
        return out
    dout, grad = st["dout"], torch.zeros_like(table, dtype=torch.float64)
    for b in range(table.shape[0]):
        here = torch.where((bucket == b).unsqueeze(-3), dout, torch.zeros_like(dout))
        sums = here.sum((-1, -2), dtype=torch.float64)
        grad[b] = sums if sums.dim() == 1 else sums.sum(0)
    return out, grad.to(st["table"].dtype)


_run_plain = {"dropout_add": _plain_add, "dropout_add_layer_norm": _plain_norm, "relative_position_bias": _plain_bias}


# ---- the work that no form can do without ------------------------------------------------------------
def work(case):
    size = {n: t.itemsize for n, t in _TYPES.items()}
    if case["op"] == "relative_position_bias":
        n = case["batch"] * case["heads"] * case["q"] * case["k"]
        table = 4 * case["heads"] * _bucket_count(case)
        moved = n * size[case["mode"]] + table
        # a comparison per pair and a sum per element
        return {"bytes": moved * (2 if case["backward"] else 1), "flops": n * (2 if case["backward"] else 1)}
    x, _, r = case["mode"].partition("/")
    n, cols = math.prod(_shape(case)), _shape(case)[-1]
    sx, sr = size[x], size[r or x]
    res = sr if case["residual"] else 0
    so = res or sx
    if case["op"] == "dropout_add":
        return {"bytes": n * (sx + res + so + so + sx), "flops": 3 * n}
    params = 2 * cols * size[case["weights"]]
    forward = n * (sx + res + sx + so) + params
    if not case["backward"]:
        return {"bytes": forward, "flops": 9 * n}
    # backward: dy, dh and the sum itself, which is not among the inputs' bytes once more; dx, dresidual
    return {"bytes": forward + n * (sx + so + so + sx + res) + 2 * params, "flops": 23 * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _exact_mask(shape, p, shared_dim, seed):
    sizes = [1 if shared_dim and i == len(shape) + shared_dim else n for i, n in enumerate(shape)]
    rows, cols = int(np.prod(sizes[:-1])), sizes[-1]
    nb = -(-cols // 8)
    index = np.arange(rows * nb, dtype=np.uint64)
    low = np.uint64(_M32)
    number = np.zeros((rows * nb, 8), np.uint64)
    for which in (0, 1):
        x = [index % np.uint64(nb), index // np.uint64(nb) & low, index // np.uint64(nb) >> np.uint64(32),
             np.full(rows * nb, which, np.uint64)]
        key = [seed % 2**32, seed // 2**32 % 2**32]
        for _ in range(10):
            left, right = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
            x = [right >> np.uint64(32) ^ x[1] ^ np.uint64(key[0]), right & low,
                 left >> np.uint64(32) ^ x[3] ^ np.uint64(key[1]), left & low]
            key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
        for i in range(8):
            half = x[i // 2] >> np.uint64(16 * (i % 2)) & np.uint64(0xFFFF)
            number[:, i] |= half << np.uint64(16 * (1 - which))
    keep = number.reshape(rows, nb * 8)[:, :cols] >= round(p * 2**32)
    return torch.from_numpy(np.ascontiguousarray(keep)).cuda().reshape(sizes)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "relative_position_bias":
        return _exact_bias(st)
    wide = {n: None if st.get(n) is None else st[n].detach().double().requires_grad_(case["backward"])
            for n in ("x", "residual", "weight", "bias")}
    update = wide["x"]
    if st["p"] > 0:
        update = update * _exact_mask(tuple(update.shape), st["p"], st["shared_dim"], st["seed"]).double() / (1 - st["p"])
    h = update if wide["residual"] is None else wide["residual"] + update
    leaves = [t for t in wide.values() if t is not None]
    if case["op"] == "dropout_add":
        return tuple(t.detach() for t in (h, *torch.autograd.grad(h, leaves, st["dout"].double())))
    var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
    y = (h - mean) * torch.rsqrt(var + 1e-5) * wide["weight"] + wide["bias"]
    if not case["backward"]:
        return y, h
    grads = torch.autograd.grad((y, h), leaves, (st["dy"].double(), st["dh"].double()))
    return tuple(t.detach() for t in (y, h, *grads))


def _exact_bucket_of(case, d):
    """The bucket of one difference key - query."""
    top, count = case["max_distance"], case["num_buckets"]
    if not count:
        return max(-top, min(top, d)) + top if case["bidirectional"] else max(0, min(top, -d))
    side = count // 2 if case["bidirectional"] else count
    first, n = side // 2, abs(d) if case["bidirectional"] else max(0, -d)
    behind = side if case["bidirectional"] and d > 0 else 0
    if n < first:
        return n + behind
    if n >= top:
        return side - 1 + behind
    wide = side - first
    j = int(math.log(n / first) / math.log(top / first) * wide)
    # (the logarithm may fall on the wrong side of a border)
    while j > 0 and n**wide < top**j * first ** (wide - j):
        j -= 1
    while j + 1 < wide and n**wide >= top ** (j + 1) * first ** (wide - j - 1):
        j += 1
    return min(first + j, side - 1) + behind


def _exact_bias(st):
    case = st["case"]
    top = case["max_distance"]
    of = np.array([_exact_bucket_of(case, d) for d in range(-top, top + 1)])
    q, k = (np.atleast_2d(t.cpu().numpy()) for t in _positions(st))
    table = st["table"].detach().double().cpu().numpy()
    H = table.shape[1]
    out, grad = [], np.zeros_like(table)
    dout = st["dout"].reshape(len(q), H, q.shape[1], k.shape[1]) if case["backward"] else None
    for b in range(len(q)):
        bucket = of[np.clip(k[b][None, :] - q[b][:, None], -top, top) + top]
        if st["groups"] is not None:
            gq, gk = (g[b].cpu().numpy() for g in st["groups"])
            bucket = np.where(gk[None, :] == gq[:, None], bucket, len(table) - 1)
        out.append(torch.from_numpy(table.T.copy()).cuda()[:, torch.from_numpy(bucket).cuda()])
        for h in range(H if case["backward"] else 0):
            grad[:, h] += np.bincount(bucket.ravel(), dout[b, h].double().cpu().numpy().ravel(), minlength=len(table))
    bias = torch.stack(out) if st["groups"] is not None or len(q) > 1 else out[0]
    return (bias, torch.from_numpy(grad).cuda()) if case["backward"] else bias
