"""Plain 64-bit forms of the paged-cache operators (numpy) and the batches their tests use."""
import numpy as np

NP = {"f32": np.float32, "f16": np.float16}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # relative rounding error of a normal value
TINY = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-134}    # half a step of the subnormals


def round_to(x, t):
    """x (float) rounded to nearest even to type t, as float64."""
    x = np.asarray(x, np.float32)
    if t == "bf16":
        b = x.view(np.uint32).astype(np.uint64)
        b = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16).astype(np.uint32)
        return b.view(np.float32).astype(np.float64)
    with np.errstate(over="ignore"):
        return x.astype(NP[t]).astype(np.float64)


def norm_rope(x, gamma, eps, cos, sin):
    """x [rows][heads][D], cos/sin [rows][r] or None: (value, what its rounding errors scale with)."""
    x = np.asarray(x, np.float64)
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gamma, np.float64)
    if cos is None:
        return x, np.abs(x)
    r = cos.shape[-1]
    c, s = (np.asarray(z, np.float64)[:, None] for z in (cos, sin))
    a, b, rest = x[..., :r], x[..., r:2 * r], x[..., 2 * r:]
    val = np.concatenate([a * c - b * s, b * c + a * s, rest], -1)
    mag = np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s), abs(rest)], -1)
    return val, mag


class Batch:
    """Sequences with new[s] new rows and len[s] positions in all, over shuffled pages."""

    def __init__(self, rng, new, total, page, spare=2, extra_rows=0, wide=None):
        self.new, self.total, self.page = list(new), list(total), page
        self.seqs = len(self.new)
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.len = np.array(self.total, np.int32)
        self.rows = int(self.start[-1]) + extra_rows
        need = [max(0, -(-t // page)) for t in self.total]
        self.pages = sum(need) + spare
        self.wide = wide or max(1, max(need))
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.seqs, self.wide), 2**31 - 1, np.int32)  # what is not read may be anything
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.free = order[at:]  # pages of no sequence

    def place(self, s, p):
        return self.table[s, p // self.page], p % self.page


def attention(b, q, kp, vp, scale, window, bad_pages=()):
    """q [rows][Hq][D], kp/vp [pages][slot][Hk][D] (float64). Returns out, lse, the sums
    sum_j w_j |v_j| and the largest scale * sum_d |q_d k_jd| of each (row, head); NaN rows
    are those that no sequence owns."""
    rows, hq, d = q.shape
    hk = kp.shape[2]
    g = hq // hk
    out, mass = np.full((rows, hq, d), np.nan), np.zeros((rows, hq, d))
    lse, size = np.full((rows, hq), np.nan), np.zeros((rows, hq))
    for s in range(b.seqs):
        n, total = b.new[s], b.total[s]
        for i in range(n):
            p, row = total - n + i, b.start[s] + i
            js = [j for j in range(max(0, p + 1 - window) if window else 0, p + 1)
                  if b.table[s, j // b.page] not in bad_pages]
            for h in range(hq):
                if not js:
                    out[row, h], lse[row, h] = 0.0, -np.inf
                    continue
                k = np.stack([kp[b.table[s, j // b.page], j % b.page, h // g] for j in js])
                v = np.stack([vp[b.table[s, j // b.page], j % b.page, h // g] for j in js])
                x = scale * (k @ q[row, h])
                m = x.max()
                w = np.exp(x - m)
                lse[row, h] = m + np.log(w.sum())
                w /= w.sum()
                with np.errstate(invalid="ignore"):
                    out[row, h] = w @ v
                    mass[row, h] = w @ np.abs(v)
                size[row, h] = scale * (np.abs(k) @ np.abs(q[row, h])).max()
    return out, lse, mass, size


def attention_bounds(b, out, mass, size, act, kv, dim):
    """How far out (and lse) may be: from the roundings the operator makes.

    A score: products of the rows' and the cache's values, exact or in two halves of 22
    bits together, summed in f32 over dim terms (the tensor cores may truncate: a whole
    step, 2^-23, per term): ds <= (dim * 2^-23 + 2^-21) * scale * sum |q k|. A weight
    exp(s - m): relative error ds, the exponential's own (a few 2^-23, taken as 2^-20), and
    its rounding to the type it is multiplied in (16-bit rows: half a step of that type;
    f32 rows: 2^-21). The same holds for the sum of the weights, so out is off by at most
    twice that times sum w|v|, then by the f32 sum over the positions (2^-23 each, twice)
    and the rounding of the result."""
    ds = (dim * 2.0**-23 + 2.0**-21) * size + 2.0**-20
    up = {"f32": 2.0**-21, "f16": 2.0**-11, "bf16": 2.0**-8}[act]
    longest = max(1, max(b.total))
    rel = 2 * (ds + up) + 2 * longest * 2.0**-23
    bound = rel[..., None] * mass * 1.01 + HALF_STEP[act] * np.abs(out) * 1.01 + 2 * TINY[act]
    return bound, ds + up + longest * 2.0**-23 + 2.0**-22 + HALF_STEP["f32"] * 64
