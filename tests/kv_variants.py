"""Batches for every kernel of the attention over the 4-bit cache: the query tiles
of an item and the warps of a CTA that the library's rule takes (kv_variant of
gollama_b200/csrc/kv_plan.h), at lengths where a warp takes several tiles of keys
and items are cut between CTAs.  tests/test_kv_variants.py says without a device
that they do, and compares them on one."""
import numpy as np

# (query tiles, warps) of a head_dim
VARIANTS = [(hd, tiles, warps) for hd in (32, 64, 96, 128)
            for tiles, warps in ((0, 4), (0, 16), (1, 4), (1, 16), (2, 4), (4, 4) if hd <= 64 else (3, 4))]


def batches(hd, tiles, warps):
    """(name, kv_heads, group, page, lens, news) of a variant: uneven lengths that make several units for each CTA,
    even ones (pieces of one item each), and short ones with empty sequences."""
    r = np.random.default_rng(hd + 10 * tiles + warps)
    uneven = lambda n, most: [int(x) for x in (most * (1 - 0.6 * r.random(n)))]  # noqa: E731
    if warps == 16:  # few items: one long beside short ones, which leave it no even pieces
        group = 4 if tiles == 0 else 7
        return [("uneven", 1, group, 48, [int(x) for x in r.integers(1, 500, 70)] + [260000], None),
                ("even", 1, group, 64, [50000] * 2, None),
                ("short", 2, group, 16, [1, 0, 511, 513, 2000], None)]
    # more items than CTAs
    if tiles < 2:  # one token each
        group = 3 if tiles == 0 else 8
        return [("uneven", 4, group, 16, uneven(155, 1300), None),
                ("even", 4, group, 32, [2048] * 24, None),
                ("short", 2, group, 16, [0, 1, 31, 33, 127, 128, 129, 300] * 5, None)]
    new, group = {2: (3, 5), 3: (5, 4), 4: (37, 8)}[tiles]
    kv_heads, seqs = {2: (4, 120), 3: (4, 80), 4: (2, 23)}[tiles]
    some = 16 if tiles < 4 else 3
    return [("uneven", kv_heads, group, 48, uneven(seqs, 1300), [new] * seqs),
            ("even", 1, group, 64, [2048] * some, [new] * some),
            ("short", 2, group, 16, [new, new + 1, 130, 400, 2], [new] * 5)]


CASES = [(*v, i) for v in VARIANTS for i in range(3)]
