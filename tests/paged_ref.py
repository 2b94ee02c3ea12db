"""The paged calls' definitions in 64 bits (numpy), the batches the tests make, and what a correct result may be off by."""
import numpy as np

U32 = 2.0 ** -24                                  # half a step of a float32, relative
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TYPES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3}


def round_to(x, kind):
    """float values rounded to a type's values (float64)"""
    import geode_amd as g

    if kind == "f32":
        return np.asarray(x, np.float32).astype(np.float64)
    t = TYPES[kind]
    return g._from_bits(g._bits16(x, t), t).astype(np.float64)


class Filled:
    """A paged cache of random contents on the device and the same values on the host. Whatever no sequence holds is
    poison: NaNs (16-bit pools), NaN scales (int8 pools)."""

    def __init__(self, seed, kind, rows, lens, page, nkv, hd, by_position=False, n_rows=None, max_len=None, spare=2,
                 first_row=0, max_rows=None):
        import geode_amd as g

        r = np.random.default_rng(seed)
        self.kind, self.rows, self.lens, self.page = kind, np.array(rows), np.array(lens), page
        self.start = np.concatenate([[0], np.cumsum(self.rows)]) + first_row
        need = -(-self.lens // page)
        pool = int(need.sum()) + spare
        order = r.permutation(pool)
        wide = max(1, int(need.max())) + 1
        self.pages = np.full((len(lens), wide), -7, np.int32)   # (entries past a length are not read)
        at = 0
        for i, n in enumerate(need):
            self.pages[i, :n] = order[at:at + n]
            at += n
        self.cache = g.PagedCache(TYPES[kind], pool, page, nkv, hd, by_position)
        self.batch = g.PagedBatch(self.rows, self.lens, self.pages, n_rows=n_rows, max_len=max_len, first_row=first_row,
                                  max_rows=max_rows)
        shape = (pool, nkv, page, hd)
        self.host = {}
        used = np.zeros((pool, page), bool)
        for i, n in enumerate(self.lens):
            for p in range(need[i]):
                used[self.pages[i, p], :max(0, min(page, n - p * page))] = True
        for name in ("k", "v"):
            if kind == "i8":
                codes = r.integers(-127, 128, shape)
                scale = np.where(used[:, None, :], r.uniform(0.5, 3.0, shape[:3]) / 127.0, np.nan).astype(np.float32)
                self.cache.write(name, codes, scale)
                self.host[name] = codes * scale[..., None].astype(np.float64)
            else:
                x = round_to(r.standard_normal(shape), kind)
                x[np.broadcast_to(~used[:, None, :], shape[:3])] = np.nan
                self.cache.write(name, x)
                self.host[name] = x

    def rewrite(self):
        """the host's values to the device again (16-bit pools)"""
        for name in ("k", "v"):
            self.cache.write(name, self.host[name])

    def place(self, i, pos):
        return self.pages[i, pos // self.page], pos % self.page

    def sequence(self, name, i):
        """[head, position, dim] of sequence i"""
        ids = self.pages[i, :-(-int(self.lens[i]) // self.page)]
        x = self.host[name][ids].transpose(1, 0, 2, 3)
        return x.reshape(x.shape[0], -1, x.shape[3])[:, :int(self.lens[i])]


def attention(f, q, scale, kind, visible=None):
    """out [row, head, dim], lse [row, head] and the largest error a correct kernel may show in each element of out and
    in lse, in 64 bits, for queries q (float64) over a Filled cache and results of type `kind`.

    The error's bound: a score is a sum of hd products of exact keys with a query of at least 21 bits, added up in fp32
    by groups of 32 (at most 4 roundings a group at the partial sum's size, itself at most A = scale sum |q k|) and
    scaled twice: ds = A (2^-21 + 4 (hd / 32 + 2) 2^-24). A weight moves by ds, by the exponential's own two steps and its
    argument's rounding (|s - m| 2^-24), and is kept to 16 bits or more for 16-bit results, 21 for fp32 ones (truncated:
    2^-15, 2^-20). The sums over positions are made of at most 8 + n / 128 steps of 4 roundings. All relative to
    W = sum p |v|; the division by the sum of weights moves out by as much again. Then the result's own rounding."""
    T, nh, hd = q.shape
    weights = 2.0 ** -20 if kind == "f32" else 2.0 ** -15
    out, lse = np.zeros((T, nh, hd)), np.full((T, nh), -np.inf)
    tol, tol_lse = np.zeros((T, nh, hd)), np.zeros((T, nh))
    for i in range(len(f.lens)):
        n, c = int(f.lens[i]), int(f.rows[i])
        if c == 0:
            continue
        k, v = f.sequence("k", i), f.sequence("v", i)
        for r in range(f.start[i], f.start[i + 1]):
            j = r - f.start[i]
            bits = (2 << j) - 1 if visible is None else int(visible[r])
            keep = np.array([p < n - c or bits >> (p - n + c) & 1 for p in range(n)], bool)
            if not keep.any():
                continue
            for h in range(nh):
                kk, vv = k[h // (nh // k.shape[0])][keep], v[h // (nh // k.shape[0])][keep]
                with np.errstate(invalid="ignore"):
                    s = kk @ q[r, h] * scale
                    m = s.max()
                    e = np.exp(s - m)
                    out[r, h] = e @ vv / e.sum()
                    lse[r, h] = m + np.log(e.sum())
                    p = e / e.sum()
                    A = (np.abs(kk) @ np.abs(q[r, h])).max() * scale
                    ds = A * (2.0 ** -21 + 4 * (hd / 32 + 2) * U32)
                    near = (m - s)[p > 2.0 ** -30].max()
                    rel = ds + 2.0 ** -22 + near * U32 + 4 * (8 + n / 128) * U32
                    W = p @ np.abs(vv)
                    tol[r, h] = W * (2 * rel + weights) + HALF_STEP[kind] * np.abs(out[r, h]) + 2.0 ** -25
                    tol_lse[r, h] = 2 * rel + U32 * (abs(lse[r, h]) + 4)
    return out, lse, tol, tol_lse
