"""Plain implementations in 64 bits that the tests of paged.py and mxfp4.py compare against, and the
error bounds that belong to them.

Tree attention, bound per output element.  With w the exact softmax weights, v the values, eps the step of
the storage type (torch.finfo(t).eps), u = 2^-24:
  * the result is rounded once: eps / 2 * |out|;
  * a weight may be rounded to the storage type before it meets v: eps / 2 * A with A = sum w |v|;
  * a score is a float32 sum of d products, times scale, times log2 e: |error| <= (d + 4) u * S with
    S = max over the keys of scale * sum |q_i k_i|; it moves the weight and the normaliser by that much
    each, exp2 adds 2 u each: 2 ((d + 4) S + 2) u * A;
  * numerator and denominator are float32 sums over n keys in some order, every partial sum rescaled by
    a rounded factor at most once per 32 keys: 2 (n + n / 16 + 8) u * A.
Products, bound per output element: a float32 sum of k exact products in any order is off by at most
k u * sum |x w| (+ the bias: one more), rounded once to the output type; GELU has a slope of at most 1.13
and its float32 evaluation adds at most 16 u |y|.
"""
import numpy as np
import torch

U = 2.0 ** -24


# ------------------------------------------------------------------------------------- paged plan
def plan_reference(cached, new, table, held, free, ring, block, rows):
    """Request by request; returns the state after the step as Python / numpy values."""
    table, free = table.copy(), free.copy()
    head, tail = int(ring[0]), int(ring[1])
    n_ring = len(free)
    starts, slots, positions, now = [0], [], [], []
    returned = []
    for i in range(len(cached)):
        have, want = int(held[i]), -(-(int(cached[i]) + int(new[i])) // block)
        for j in range(have, want):
            table[i, j] = free[head % n_ring]
            head += 1
        returned += [int(table[i, j]) for j in range(want, have)]
        now.append(want)
        for p in range(int(cached[i]), int(cached[i]) + int(new[i])):
            positions.append(p)
            slots.append(int(table[i, p // block]) * block + p % block)
        starts.append(starts[-1] + int(new[i]))
    for b in returned:
        free[tail % n_ring] = b
        tail += 1
    pad = [-1] * (rows - starts[-1])
    return dict(table=table, free=free, held=np.array(now), ring=np.array([head, tail]), starts=np.array(starts),
                slots=np.array(slots + pad), positions=np.array(positions + pad))


# ---------------------------------------------------------------------------------- tree attention
def tree_paths(parents, n):
    """seen[a][b]: is b on the path from a to its root (parents outside [0, a) are roots)."""
    seen = np.zeros((n, n), dtype=bool)
    for a in range(n):
        p = a - 1 if parents is None else int(parents[a])
        if 0 <= p < a:
            seen[a] = seen[p]
        seen[a, a] = True
    return seen


def tree_reference(q, k, v, k_cache, v_cache, table, cached, starts, slots, parents, scale=None):
    """(out, bound, k_cache, v_cache): attention in float64 and its error bound, the caches after the store.
    Rows outside every sequence are NaN in `out`.  All tensors on the CPU."""
    rows, heads, d = q.shape
    n_blocks, kv, block, _ = k_cache.shape
    group = heads // kv
    scale = d ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    out = torch.full((rows, heads, d), float("nan"), dtype=torch.float64)
    bound = torch.zeros((rows, heads, d), dtype=torch.float64)
    kd, vd, qd = k.double(), v.double(), q.double()
    for i in range(len(cached)):
        lo, hi = int(starts[i]), int(starts[i + 1])
        n = hi - lo
        if n == 0:
            continue
        at = [p for p in range(min(int(cached[i]), table.shape[1] * block))
              if 0 <= int(table[i, p // block]) < n_blocks]
        blk = torch.tensor([int(table[i, p // block]) for p in at], dtype=torch.long)
        off = torch.tensor([p % block for p in at], dtype=torch.long)
        hk, hv = k_cache[blk, :, off].double(), v_cache[blk, :, off].double()         # [c, kv, d]
        seen = tree_paths(None if parents is None else parents[lo:hi], n)
        for a in range(n):
            mine = torch.from_numpy(np.nonzero(seen[a])[0])
            keys = torch.cat([hk, kd[lo:hi][mine]])
            vals = torch.cat([hv, vd[lo:hi][mine]])
            for h in range(heads):
                kk, vv = keys[:, h // group], vals[:, h // group]
                z = kk @ qd[lo + a, h] * scale
                w = torch.softmax(z, dim=0)
                o, big = w @ vv, w @ vv.abs()
                s = float((kk.abs() @ qd[lo + a, h].abs()).max()) * abs(scale)
                c = len(z)
                out[lo + a, h] = o
                bound[lo + a, h] = eps / 2 * o.abs() + (eps / 2 + 2 * ((d + 4) * s + 2) * U + 2 * (c + c / 16 + 8) * U) * big
    kc, vc = k_cache.clone(), v_cache.clone()
    for r in range(rows):
        s = int(slots[r])
        if 0 <= s < n_blocks * block and any(int(starts[i]) <= r < int(starts[i + 1]) for i in range(len(cached))):
            kc[s // block, :, s % block], vc[s // block, :, s % block] = k[r], v[r]
    return out, bound, kc, vc


# ------------------------------------------------------------------------------------------- mxfp4
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize_reference(x):
    """(codes [rows, k] 0..15, scale bytes [rows, k / 32]) of a float64 matrix, by the definition: the nearest
    value of the grid, at equal distance the one with the even code."""
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    top = np.abs(b).max(axis=2)
    with np.errstate(all="ignore"):
        e = np.where(top > 0, np.frexp(np.where(np.isfinite(top), top, 1.0))[1] - 1 - 2, -127)
    e = np.clip(e, -127, 127)
    dist = np.abs(np.abs(np.ldexp(np.where(np.isfinite(b), b, 0.0), -e[..., None]))[..., None] - GRID)
    best = dist.min(axis=-1, keepdims=True)
    even_first = np.array([0, 2, 4, 6, 1, 3, 5, 7])
    code = even_first[np.argmax((dist == best)[..., even_first], axis=-1)]
    code = code + 8 * np.signbit(b)
    scales = (e + 127).astype(np.uint8)
    bad = ~np.isfinite(b).all(axis=2)
    scales[bad] = 255
    return code.reshape(rows, k).astype(np.uint8), scales


def values_of(codes, scales):
    """float64 values of unpacked codes [rows, k] under scale bytes [rows, k / 32]."""
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(s, 32, axis=1)


def unpack(codes):
    """[rows, k / 2] bytes -> [rows, k] codes (element 2 i in the low half)."""
    return np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[0], -1)


def gelu_reference(y, kind):
    if kind == "tanh":
        return 0.5 * y * (1 + torch.tanh((2 / np.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    if kind == "erf":
        return 0.5 * y * (1 + torch.erf(y / 2 ** 0.5))
    return y


def product_reference(x, w, bias, gelu, out_dtype):
    """(y, bound) in float64 of act(x w^T + bias); x, w float64."""
    y, mass = x @ w.t(), x.abs() @ w.abs().t()
    k = x.shape[1]
    if bias is not None:
        y, mass = y + bias.double(), mass + bias.double().abs()
    err = (k + 1) * U * mass
    z = gelu_reference(y, gelu)
    if gelu:
        err = 1.13 * err + 16 * U * y.abs()
    return z, err + torch.finfo(out_dtype).eps / 2 * (z.abs() + err)
