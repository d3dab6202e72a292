"""Cases of the attention over a part of the KV cache whose results are held to a 2-norm: T, pos0, query heads, KV heads, dims, window,
sinks. Where more than about a thousand keys are seen they are split over waves and workgroups, so that the bound lies below what a
lost piece of a weight changes."""
import numpy as np

import span_ref as ref

CHAIN = 1024                                # keys that one wave adds up, at most: more of them are split over waves and workgroups

NORM_WINDOWS = [
    # a column a 32-dim group; a column a row (more rows of a KV head than fit so); one token and a few
    (1, 4095, 16, 8, 128, 1024, 4), (1, 300, 40, 8, 96, 170, 3), (1, 2500, 16, 1, 32, 2000, 64), (1, 900, 20, 1, 128, 500, 7), (1, 700, 64, 2, 64, 4096, 5),
    (1, 6000, 16, 8, 128, -1, 0), (1, 20000, 8, 8, 128, 15000, 100), (1, 1000, 8, 8, 64, 999, 1),
    (3, 1000, 32, 16, 64, 100, 100), (5, 700, 6, 6, 96, 333, 2), (8, 4000, 16, 16, 128, 512, 4), (2, 1500, 8, 2, 128, 700, 33), (4, 640, 12, 6, 32, 65, 5),
    # more rows: ranges of keys that are merged, and one range
    (16, 700, 1, 1, 128, 160, 0), (17, 600, 3, 3, 64, -1, 9), (65, 130, 5, 5, 64, 64, 0), (64, 1000, 16, 8, 128, 900, 0), (100, 150, 6, 2, 96, 31, 40),
    (130, 17, 8, 4, 32, 120, 16), (257, 0, 4, 2, 128, 64, 4), (300, 5, 20, 1, 32, 77, 1), (700, 64, 4, 4, 96, -1, 0), (513, 400, 4, 1, 128, 300, 65),
]


def inputs(T, pos0, nHq, nKv, hd):
    """Queries of the size that normalised heads have, and a cache: scores of about one, so that every key counts for something."""
    rng = np.random.default_rng(7 * T + pos0 + hd)
    return rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, pos0 + T, nKv, hd)
