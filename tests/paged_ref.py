"""64-bit references of rotary positions and the paged cache, and helpers of
their tests.

Bounds.  u = 2^-24 is half a step of fp32.  Rotary: the angle is reduced in 64
bits to |y| <= pi / 4, which is rounded to fp32, multiplied by pi / 2 (rounded
itself) and rounded again: 3 u |y| < 2.4 u; the polynomials of sine and cosine
lose 2 u of 1 at most and leave out 2^-27; with the factor `scale` and its
rounding each is within 6 u |scale|.  A product and a fused multiply-add of two
values x1, x2 add 2 u: in all 8 u |scale| (|x1| + |x2|), and the angle's own 64
bits |a| 2^-51.  What enters a bf16 cache is rounded once more, by 2^-8 of it.
"""
import numpy as np

U = 2.0 ** -24


def to_bf16(x):
    """float32 rounded to bf16, to the nearest, ties to even (finite or infinite values), as uint16."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(h):
    return (np.asarray(h, np.uint16).astype(np.uint32) << 16).view(np.float32)


def frequencies(rot, base=10000.0):
    return (base ** (-2.0 * np.arange(rot // 2) / max(rot, 2))).astype(np.float32)


def rotary(x, positions, freq, rot, layout, scale=1.0, back=False):
    """(y, bound) of x [..., dim] with positions broadcasting over x's leading dims."""
    x = np.asarray(x, np.float64)
    y, bound = x.copy(), np.zeros_like(x)
    a = np.asarray(positions, np.float64)[..., None] * np.asarray(freq, np.float64)[:rot // 2]
    s, c = np.sin(a) * (-1 if back else 1), np.cos(a)
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    p, q = x[..., one], x[..., two]
    scale = float(np.float32(scale))
    y[..., one], y[..., two] = scale * (p * c - q * s), scale * (p * s + q * c)
    bound[..., one] = bound[..., two] = abs(scale) * (np.abs(p) + np.abs(q)) * (8 * U + np.abs(a) * 2.0 ** -51)
    return y, bound


class Strided:
    """A tensor inside a larger device buffer at element strides of its leading dims (the last is contiguous)."""

    def __init__(self, ctx, values, strides=None, bf16=False):
        self.values = np.asarray(values)
        shape = self.values.shape
        if strides is None:
            strides = [int(np.prod(shape[i + 1:])) for i in range(len(shape) - 1)]
        self.strides = tuple(strides)
        index = np.arange(shape[-1])
        for n, s in zip(shape[:-1], self.strides):
            index = index[None]
        for axis, (n, s) in enumerate(zip(shape[:-1], self.strides)):
            grid = [1] * len(shape)
            grid[axis] = n
            index = index + (np.arange(n, dtype=np.int64) * s).reshape(grid)
        self.index, self.bf16 = index, bf16
        size = int(index.max()) + 1 if index.size else 1
        self.size = size + (size % 2 if bf16 else 0)
        host = np.full(self.size, 0x4442 if bf16 else 777.0, np.uint16 if bf16 else np.float32)
        host[index] = self.values
        self.host = host
        self.buf = ctx.to_device(host.view(np.float32))

    @property
    def ptr(self):
        return self.buf.ptr

    def read(self):
        """The tensor, after checking that nothing between its rows was written."""
        now = self.buf.download().view(self.host.dtype)
        keep = np.ones(now.size, bool)
        keep[self.index] = False
        assert np.array_equal(now[keep].view(np.uint8), self.host[keep].view(np.uint8)), "written outside the tensor"
        return now[self.index]


class Ints:
    """An int32 device array."""

    def __init__(self, ctx, values):
        self.buf = ctx.to_device(np.ascontiguousarray(values, np.int32).view(np.float32))

    def set(self, values):
        self.buf.upload(np.ascontiguousarray(values, np.int32).view(np.float32))

    @property
    def ptr(self):
        return self.buf.ptr


class Pool:
    """Pages of sequences of given lengths, handed out in random order; unused slots hold NaN.

    k, v: [pages, kv_heads, page_size, dim] float32 (for a bf16 cache: values that bf16 holds)."""

    def __init__(self, seed, lens, kv_heads, page, dim, dtype="f32", order="phsd", spare=2, max_pages=None):
        rng = np.random.default_rng(seed)
        self.lens, self.kv_heads, self.page, self.dim, self.dtype = list(lens), kv_heads, page, dim, dtype
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        self.max_pages = max(max(need, default=0), 1) if max_pages is None else max_pages
        ids = rng.permutation(self.pages)
        # entries past a sequence's length are not read: any number may stand there
        self.table = np.full((len(lens), self.max_pages), 0x7FFFFFF0, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.k, self.v = (np.full((self.pages, kv_heads, page, dim), np.nan, np.float32) for _ in range(2))
        for b, n in enumerate(lens):
            j = np.arange(n)
            for t in (self.k, self.v):
                x = rng.standard_normal((n, kv_heads, dim)).astype(np.float32)
                t[self.table[b, j // page], :, j % page] = from_bf16(to_bf16(x)) if dtype == "bf16" else x
        self.order = order

    def strides(self):
        h, s, d = self.kv_heads, self.page, self.dim
        if self.order == "phsd":
            return (h * s * d, s * d, d)
        if self.order == "pshd":
            return (s * h * d, d, h * d)
        return (h * (s * (d + 3) + 5) + 7, s * (d + 3) + 5, d + 3)  # gaps

    def place(self, ctx):
        """The cache on the device."""
        from zigneuron_amd import PagedCache
        bf = self.dtype == "bf16"
        raw = (lambda t: np.where(np.isnan(t), np.uint16(0x7FC0), to_bf16(np.nan_to_num(t)))) if bf else (lambda t: t)
        self.dk, self.dv = (Strided(ctx, raw(t), self.strides(), bf) for t in (self.k, self.v))
        self.dtable, self.dlens = Ints(ctx, self.table), Ints(ctx, self.lens)
        return PagedCache(self.dk.ptr, self.dv.ptr, self.dtable.ptr, self.dlens.ptr, len(self.lens), self.pages, self.page,
                          self.max_pages, self.kv_heads, self.dim, self.dtype, self.strides())

    def read(self):
        """k and v as float32."""
        return tuple(from_bf16(t.read()) if self.dtype == "bf16" else t.read() for t in (self.dk, self.dv))

    def dense(self, b, k=None, v=None, keep=None):
        """Sequence b's keys and values [1, kv_heads, positions, dim], of the positions in keep (None: all)."""
        js = np.arange(self.lens[b]) if keep is None else np.asarray(keep, int)
        pages = self.table[b, js // self.page]
        return tuple(t[pages, :, js % self.page].transpose(1, 0, 2)[None] for t in (self.k if k is None else k, self.v if v is None else v))


def starts_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
