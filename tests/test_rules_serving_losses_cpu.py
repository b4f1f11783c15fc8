"""The dispatch rules of the serving operators at more sizes where both sides were timed on the card, the slower side
included: what a rule loses there, and no more than that."""
from test_rules_cpu import _run

# The adapters' rule sees rows and columns, not which rows share an adapter: ids are device memory. Wide tiles multiply
# all their rows by each of their adapters, so many adapters in turn cost them more than runs of one.
ADAPTERS = [  # rows, columns, adapters, rows in a run of one, us wide, us narrow
    (1000, 6144, 24, 1, 82.1, 70.6), (1000, 6144, 8, 1, 47.5, 49.0), (1000, 6144, 24, 40, 24.3, 27.8), (500, 6144, 8, 1, 30.7, 32.5),
    (500, 6144, 24, 1, 53.1, 48.6), (2000, 6144, 24, 1, 133.3, 134.0), (4000, 6144, 24, 1, 242.2, 248.2), (4000, 2560, 8, 1, 236.3, 268.2),
    (4000, 2560, 24, 1, 419.1, 436.5), (2000, 19456, 16, 1, 248.5, 280.0), (2000, 19456, 24, 1, 296.7, 304.4),
    (1000, 2560, 24, 1, 149.7, 141.8), (1000, 2560, 8, 1, 81.0, 88.1), (600, 2560, 2, 1, 13.5, 13.4), (250, 6144, 8, 1, 19.6, 17.7),
    (300, 6144, 24, 1, 35.6, 31.2), (300, 6144, 4, 1, 15.4, 16.7), (100, 19456, 24, 1, 31.1, 26.9), (80, 19456, 8, 1, 17.6, 16.2),
    (100, 19456, 4, 1, 16.2, 16.7), (200, 19456, 24, 1, 45.9, 40.2), (200, 19456, 4, 1, 24.2, 23.5), (1500, 1024, 24, 1, 104.2, 104.8),
    (200, 2560, 24, 1, 62.4, 36.5),
]
SLOWER = {(1000, 6144, 24, 1), (500, 6144, 24, 1), (1000, 2560, 24, 1), (250, 6144, 8, 1), (300, 6144, 24, 1), (100, 19456, 24, 1),
          (80, 19456, 8, 1), (200, 19456, 24, 1)}  # by more than 5 %: the wide side taken

ATTENTION = [  # KV heads and sequences, rows of each, keys, values of a head, F32 y, us 16 rows a workgroup, us many
    (8, 128, 2064, 256, 1, 35.1, 37.0), (8, 128, 2064, 256, 0, 31.1, 30.2), (8, 4096, 2048, 256, 1, 356.9, 231.7),
    (8, 4096, 2048, 256, 0, 282.8, 115.9), (64, 512, 128, 256, 1, 79.8, 33.9), (64, 512, 128, 256, 0, 69.5, 22.6),
    (8, 1024, 512, 256, 1, 39.5, 41.2), (8, 1024, 512, 256, 0, 33.0, 32.6), (8, 514, 387, 256, 1, 32.2, 39.9), (8, 514, 387, 256, 0, 27.2, 33.0),
    (64, 64, 4016, 256, 1, 95.9, 127.3), (64, 64, 4016, 256, 0, 76.7, 68.5), (8, 128, 464, 256, 1, 20.7, 29.3), (8, 128, 464, 256, 0, 19.3, 23.4),
    (8, 2048, 1024, 256, 1, 110.0, 79.7), (8, 2048, 1024, 256, 0, 89.0, 49.3), (24, 400, 600, 256, 1, 65.1, 55.1), (24, 400, 600, 256, 0, 54.3, 37.9),
    (8, 2048, 1024, 128, 1, 56.2, 47.2), (8, 2048, 1024, 128, 0, 47.6, 35.0), (8, 1024, 512, 128, 1, 21.8, 35.0), (8, 1024, 512, 128, 0, 19.5, 25.2),
    (64, 64, 4016, 128, 1, 54.2, 91.2), (64, 64, 4016, 128, 0, 45.5, 39.2), (8, 4096, 2048, 64, 1, 110.7, 72.0), (8, 4096, 2048, 64, 0, 94.3, 52.2),
    (64, 64, 4016, 64, 1, 38.2, 42.4), (64, 64, 4016, 64, 0, 33.1, 30.6), (8, 1024, 512, 64, 1, 14.0, 24.2), (8, 1024, 512, 64, 0, 13.1, 21.0),
]


def _losses(rows, got):
    """What the side taken (true: the last but one time, wide; for attention the last, many) takes over the other."""
    return [(a if g else b) / min(a, b) for (a, b), g in zip(rows, got)]


def test_adapters(tmp_path):
    got = _run(tmp_path, lambda r: f"lora_wide({r[0]}, {r[1]})", ADAPTERS)
    loss = _losses([r[4:6] for r in ADAPTERS], got)
    assert {r[:4] for r, x in zip(ADAPTERS, loss) if x > 1.05} == SLOWER
    assert max(loss) < 1.17
    # where the rows of a tile have one adapter, and at up to 8 adapters in turn, it loses 11 % at most
    assert max(x for r, x in zip(ADAPTERS, loss) if r[2] <= 8 or r[3] > 16) < 1.11


def test_attention(tmp_path):
    got = _run(tmp_path, lambda r: f"fa4_plan({r[0]}, {r[1]}, {r[2]}, {r[3]}, {r[4]}, false, 256).many", ATTENTION)
    loss = _losses([(r[6], r[5]) for r in ATTENTION], got)
    assert {r[:5] for r, x in zip(ATTENTION, loss) if x > 1.06} == {(64, 64, 4016, 64, 1)}  # short rows of 64 values in F32
    assert max(loss) < 1.12
