"""A paged KV cache in 8 bits, in plain numpy: rows as int8 and a scale, pools as the handle lays them out, and the batch of
test_gpu_paged.Case on such pools."""
import numpy as np

from tests.test_gpu_paged import Case


def held(x):
    """(q, scale) of rows [.., hd] of fp32: scale = max |x| / 127 in fp32, q = x / scale to the nearest whole number, half away from
    zero, decided exactly (a quotient's distance from a half is at least 2^-33 of it where it is not 0, far more than 64 bits lose); a row with a
    value that is no number: q 0, scale NaN."""
    x = np.asarray(x, np.float32)
    odd = ~np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        scale = np.abs(x).max(-1) / np.float32(127)
        assert scale.dtype == np.float32
        size = np.abs(x.astype(np.float64))
        n = np.minimum(np.floor(size / scale[..., None].astype(np.float64) + 0.5), 127)
    q = np.where((scale > 0)[..., None] & ~odd[..., None], np.sign(x) * np.nan_to_num(n), 0).astype(np.int8)
    return q, np.where(odd, np.float32(np.nan), scale)


def values(q, scale):
    """What rows [.., kv, hd] stand for, in 64 bits."""
    return q.astype(np.float64) * scale.astype(np.float64)[..., None]


def pool(q, scale, page):
    """The bytes of a pool: rows [slots, kv, hd], then scales [pages, kv, page]."""
    n, kv = scale.shape
    return np.concatenate([np.ascontiguousarray(a).reshape(-1).view(np.uint8) for a in (q, scale.reshape(n // page, page, kv).transpose(0, 2, 1))])


def from_pool(data, slots, kv, hd, page):
    data = np.asarray(data, np.uint8)
    q, s = data[:slots * kv * hd].view(np.int8), data[slots * kv * hd:].view(np.float32)
    return q.reshape(slots, kv, hd).copy(), s.reshape(slots // page, kv, page).transpose(0, 2, 1).reshape(slots, kv).copy()


class Case8(Case):
    """A batch over Q8 pools.  What no request holds has any whole numbers, and NaN for its scale."""

    def __init__(self, hip, bufs, heads, kv, hd, page, new, lens, seed=0, **more):
        super().__init__(hip, bufs, heads, kv, hd, 8, page, new, lens, seed=seed, **more)
        self.q8, self.scales = {}, {}
        for name in ("K", "V"):
            self.set_rows(name, getattr(self, name).astype(np.float32))

    def set_rows(self, name, x):
        """Quantizes fp32 rows [slots, kv * hd] (NaN: any q, scale NaN) and takes the values that they then stand for."""
        x = np.asarray(x, np.float32).reshape(-1, self.kv, self.hd)
        q, s = held(x)
        odd = np.isnan(s)
        q[odd] = self.rng.integers(-128, 128, (int(odd.sum()), self.hd))
        self.q8[name], self.scales[name] = q, s
        setattr(self, name, values(q, s).reshape(-1, self.kv * self.hd))

    def bytes_of(self, name):
        return pool(self.q8[name], self.scales[name], self.page)

    def want(self, *what, **more):
        """The bound has a term more.  A value may be a zero exactly, at the position that has nearly all of a row's weight, and then the element
        is made of weights that two fp16 terms cut off: with d_j the scales, weights p_j d_j are held times a power of two that puts the
        largest of them since the row's maximum moved last at 2^11 or more, in steps of 2^-24.  Each of a row's n is therefore off by at most
        2^-25 / 2^11 of the largest, which is at most sum_j p_j d_j, and counts with a whole number up to 127."""
        out, bound = super().want(*what, **more)
        V = self.V
        self.V = np.repeat(np.nan_to_num(self.scales["V"]).astype(np.float64), self.hd, 1)
        most, _ = super().want(*what, **more)
        self.V = V
        n = np.repeat(self.lens, self.new)[:, None].astype(np.float64)
        return out, bound + 127 * n * 2.0 ** -36 * most

    def upload(self):
        up = self.b.up
        self.out0 = np.full((max(self.bound, 1), self.ldo), 7.25, np.float32)
        assert self.h.PoolBytes() == self.bytes_of("K").size
        self.d = {"q": up(self.q), "K": up(self.bytes_of("K")), "V": up(self.bytes_of("V")), "table": up(self.table), "rowStart": up(self.rowStart),
                  "lens": up(self.lens), "out": up(self.out0)}
