"""Calls of the attention over a paged cache that reach each of its kernels: every number of query rows, cache type, width of heads and
kind of pages, with sequences of other numbers of rows beside them."""

DIMS = ((27, 32), (50, 64), (76, 96), (113, 128))  # of each width that kernels are built for


def _shapes(kernel, dtype, dim):
    """(lens, counts, group, kv_heads) of calls that `kernel` takes."""
    if kernel == "few":  # to 16 rows
        return [([150, 40, 7, 300], [3, 1, 0, 2], 4, 2), ([500], [1], 16, 1)]
    if kernel == "few2":  # 17 to 32
        return [([150, 40, 300], [5, 1, 4], 5, 2), ([700, 33], [32, 9], 1, 3)]
    if kernel == "few4":  # 33 to 64, where there are many sequences' heads
        heads = 64 if dtype == "bf16" or dim <= 64 else 256
        kv, batch = (2, heads // 2) if heads == 64 else (8, heads // 8)
        counts = [[9, 8, 1, 0, 7][i % 5] for i in range(batch)]
        one = ([700 if i == 5 else 9 + 7 * i % 60 for i in range(batch)], counts, 5, kv)
        return [one, ([64 + i % 40 for i in range(batch)], [64 - 21 * (i % 3) for i in range(batch)], 1, kv),
                ([1 + 5 * i % 90 for i in range(batch)], [1] * batch, 33, kv)]
    if kernel == "tile":
        return [([200, 150, 90], [60, 1, 3], 4, 2), ([260, 130], [260, 129], 1, 2)]
    return [([1000, 600, 700], [100, 1, 100], 4, 8)]  # wide


def cases():
    """(kernel's name, lens, counts, q heads, kv heads, page, dim, dtype)"""
    out = []
    for dtype in ("f32", "bf16"):
        for w, dims in enumerate(DIMS):
            for kernel in ("few", "few2", "few4", "tile", "wide")[:5 if dtype == "f32" else 4]:
                for i, (page, suffix) in enumerate(((24, ""), (32, "_p"), (13, ""), (16, "_p"))):
                    dim = dims[page in (13, 16)]
                    shapes = _shapes(kernel, dtype, dim)
                    # either kind of pages gets both of two shapes
                    lens, counts, group, kv = shapes[(i + w) % 3 if len(shapes) == 3 else (0, 1, 1, 0)[i] % len(shapes)]
                    out.append((f"zn_paged_{kernel}_{dtype}_{32 * w + 32}{suffix}", lens, counts, group * kv, kv, page, dim, dtype))
    return out
