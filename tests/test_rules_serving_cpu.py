"""The dispatch rules of the serving operators at sizes where both sides were timed on the card: the
quicker side is taken (sizes within 5 % of each other are left to the rule)."""
from test_rules_cpu import _run

LOGITS = [  # rows, tokens, us in tiles of 2048, of 4096
    (8, 151669, 6.0, 6.8), (64, 151669, 19.5, 18.5),
]

ADAPTERS = [  # rows, columns, us wide, us narrow
    (32, 6144, 14.5, 10.1), (64, 6144, 16.5, 11.7), (100, 6144, 17.1, 13.9), (200, 6144, 19.6, 16.7), (500, 6144, 30.7, 34.1),
    (100, 19456, 13.1, 14.9), (200, 19456, 18.1, 20.7), (200, 2560, 62.9, 36.0), (4000, 2560, 238.1, 268.4), (2000, 19456, 248.5, 290.6),
    (600, 2560, 12.9, 14.6), (4000, 1024, 24.7, 30.2), (150, 19456, 39.9, 50.2), (80, 19456, 10.8, 12.4),
]

ATTENTION = [  # KV heads and sequences, rows of each, keys, values of a head, F32 y, us 16 rows a workgroup, us many
    (8, 66, 33, 128, 1, 9.9, 19.4), (8, 66, 33, 128, 0, 9.4, 15.2), (8, 128, 464, 128, 1, 13.3, 22.8), (8, 128, 464, 128, 0, 12.5, 18.8),
    (8, 514, 387, 128, 1, 18.9, 35.4), (8, 514, 387, 128, 0, 16.8, 24.2), (8, 1024, 512, 128, 1, 23.5, 34.8),
    (8, 1024, 512, 128, 0, 20.9, 26.3), (8, 2048, 1024, 128, 1, 64.9, 50.6), (8, 2048, 1024, 128, 0, 52.3, 36.9),
    (8, 4096, 2048, 128, 1, 208.0, 98.1), (8, 4096, 2048, 128, 0, 146.5, 58.3), (64, 64, 4016, 128, 1, 58.6, 96.2),
    (64, 64, 4016, 128, 0, 47.7, 39.8), (64, 256, 4064, 128, 1, 194.8, 107.8), (64, 256, 4064, 128, 0, 147.1, 66.0),
    (64, 512, 128, 128, 1, 44.7, 28.2), (64, 512, 128, 128, 0, 35.0, 16.9), (64, 1028, 257, 128, 1, 126.8, 52.3),
    (8, 1024, 8256, 128, 1, 193.2, 112.4), (24, 400, 600, 64, 0, 19.8, 25.1), (24, 400, 600, 64, 1, 27.1, 36.6),
    (8, 514, 387, 64, 1, 12.8, 33.0), (64, 512, 128, 64, 0, 25.7, 13.9), (64, 256, 4064, 64, 1, 129.6, 73.6),
    (8, 4096, 2048, 256, 0, 288.8, 117.5), (64, 512, 128, 256, 1, 84.6, 34.0), (64, 512, 128, 256, 0, 75.3, 22.3),
    (8, 514, 387, 256, 1, 33.1, 41.2), (8, 514, 387, 256, 0, 27.1, 34.5), (24, 400, 600, 256, 0, 58.0, 37.8), (24, 400, 600, 256, 1, 68.2, 55.4),
    (64, 64, 4016, 256, 0, 79.8, 68.7), (64, 64, 4016, 256, 1, 98.9, 127.3), (8, 128, 464, 256, 1, 20.9, 29.2), (8, 128, 464, 256, 0, 19.7, 23.2),
    (8, 80, 5040, 256, 1, 46.2, 42.4), (8, 80, 5040, 256, 0, 39.8, 32.1), (8, 2048, 1024, 256, 1, 113.5, 82.3),
]

SPLITS = [  # KV heads and sequences, rows of each, keys, least and most splits that came within 12 % of the best
    (8, 2, 257, 1, 1), (8, 2, 513, 2, 3), (8, 2, 700, 2, 4), (64, 4, 512, 1, 1), (64, 4, 6600, 6, 12), (512, 4, 1501, 1, 2),
    (8, 128, 2064, 3, 9), (8, 1024, 512, 1, 1), (8, 514, 387, 1, 1),
]


def test_logits_take_the_quicker_tiles(tmp_path):
    got = _run(tmp_path, lambda r: f"logits_small_tiles({r[0]}, {r[1]}, 256)", LOGITS)
    assert got == [int(r[2] < r[3]) for r in LOGITS]


def test_adapters_take_the_quicker_tiles(tmp_path):
    got = _run(tmp_path, lambda r: f"lora_wide({r[0]}, {r[1]})", ADAPTERS)
    bad = [r for r, g in zip(ADAPTERS, got) if g != (r[2] < r[3])]
    assert not bad, bad


def test_attention_takes_the_quicker_kernel(tmp_path):
    got = _run(tmp_path, lambda r: f"fa4_plan({r[0]}, {r[1]}, {r[2]}, {r[3]}, {r[4]}, false, 256).many", ATTENTION)
    bad = [r for r, g in zip(ATTENTION, got) if g != (r[6] < r[5])]
    assert not bad, bad


def test_attention_splits_where_it_pays(tmp_path):
    got = _run(tmp_path, lambda r: f"fa4_plan({r[0]}, {r[1]}, {r[2]}, 128, true, {int(r[1] < 16)}, 256).splits", SPLITS)
    bad = [(r, g) for r, g in zip(SPLITS, got) if not r[3] <= g <= r[4]]
    assert not bad, bad


def test_attention_plans_stay_in_range(tmp_path):
    """One workgroup per compute unit or fewer, the longest rows, one row and one key."""
    rows = [(h, r, n, d, f) for h in (1, 8, 65535) for r in (1, 33, 1 << 20) for n in (1, 1 << 27) for d in (64, 128, 256) for f in (0, 1)]
    got = _run(tmp_path, lambda r: f"fa4_plan({r[0]}, {r[1]}, {r[2]}, {r[3]}, {r[4]}, false, 256).splits", rows)
    assert all(g >= 1 for g in got) and all(g == 1 for r, g in zip(rows, got) if r[2] == 1)
