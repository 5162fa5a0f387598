"""Host-side arithmetic of the feed-forward operators' matrix products, in C++ programs built from the library's own headers."""

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def build(tmp_path, source):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = tmp_path / Path(source).stem
    b = subprocess.run(["g++", "-O1", "-std=c++17", "-I", str(ROOT / "vtc_amd" / "csrc"), str(ROOT / "tests" / source), "-o", str(exe)],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-2000:]
    return exe


def halves(columns, tile, most=128):
    """First columns of the half-tiles of a product's last tile."""
    last = (columns - 1) // tile * tile
    return [last] if tile <= most else [last, last + 128]


def test_operand_windows_stay_inside_the_operand(tmp_path):
    """Every K-tile of dx (two segments, 192-wide tiles) and of the weights' gradients (256-wide tiles, long contractions), also where
    the second half of the last tile lies wholly behind the matrix and at K-tiles whose row offsets pass 2^31 bytes."""
    lines = []
    # dx: contraction over `inner`, columns of the width; K-tiles of both segments run on a half that has no columns
    for width, inner in ((16384, 53248), (768, 2048), (389, 1031), (8, 8), (1, 1), (100, 262144), (262144, 262144), (200000, 100000), (4096 + 64, 262144)):
        pitch = (width + 7) // 8 * 8
        for ld in (pitch, 1 << 20):
            for c0 in halves(width, 192):
                tiles = 2 * ((inner + 63) // 64)
                lines.append((inner, ld, width, c0, 128, (tiles + 1) & ~1, 2))
            lines.append((inner, ld, width, (width - 1) // 64 * 64, 64, 2 * ((inner + 63) // 64), 2))
    # the weights' gradients: contraction over the rows, columns of `inner`, of the width or of the output
    for rows, columns in ((78400, 13696), (200000, 13696), (2 ** 31 - 256, 8), (1_000_003, 4104), (31936, 2048), (1237, 389), (1, 1), (2 ** 24 + 1, 65)):
        pitch = (columns + 7) // 8 * 8
        for ld in (pitch, 1 << 20):
            for c0 in halves(columns, 256):
                lines.append((rows, ld, columns, c0, 128, ((rows + 63) // 64 + 1) & ~1, 1))
            lines.append((rows, ld, columns, (columns - 1) // 64 * 64, 64, (rows + 63) // 64, 1))
    exe = build(tmp_path, "op_extent_walk.cpp")
    r = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, x)) for x in lines), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    assert f"{len(lines)} products walked" in r.stdout


def plans(tmp_path, questions):
    exe = build(tmp_path, "op_plan_table.cpp")
    r = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, q)) for q in questions), capture_output=True, text=True, timeout=300)
    lines = r.stdout.splitlines()
    assert r.returncode == 0 and len(lines) == len(questions), r.stdout[-500:] + r.stderr[-500:]
    return [line.split() for line in lines]


def test_no_launch_takes_2_to_the_32_threads(tmp_path):
    most = 2 ** 24 - 1   # blocks of 256 threads
    widths = (1, 8, 64, 65, 100, 128, 129, 192, 2048, 262144)
    ask = []
    for m in (65, 10 ** 6, 2 ** 30 + 1, 2 ** 31 - 256):
        for n in widths:
            if (m // 128 + 1) * (n // 32 + 1) > 2 ** 30:   # refused as too many
                continue
            for k in (1, 64, 2048):
                ask += [("gate", m, k, n, 0), ("gate", m, k, n, 1), ("rows", m, n, k), ("dgate", m, k, n), ("weights", m, k, n, n)]
    for q, (_, _, _, blocks) in zip(ask, plans(tmp_path, ask)):
        assert 1 <= int(blocks) <= most, q
    ask = [("rotary", t, per, table) for t in (1, 7, 5000, 2 ** 24 - 1, 2 ** 24, 2 ** 25 + 3, 2 ** 26) for per, table in ((1, 2048), (24 * 4, 64), (1000, 8), (5000, 8))]
    for q, (n, blocks) in zip(ask, plans(tmp_path, ask)):
        assert 1 <= int(n) <= q[3] and int(blocks) <= most, q


def test_feed_forward_sizes_of_the_gpu_tests_cover_both_tilings(tmp_path):
    """The sizes that tests/test_ops.py checks against 64 bits: all products on small tiles, and all products on 256-wide ones.  A change of
    the cost model that moves them has to bring other sizes."""
    from test_ops import FFN_SIZES, FFN_SPLIT_SIZES, FFN_WIDE_SIZES

    def ask(m, k, f, n):
        both = 2 * 64 * ((f + 63) // 64)   # dx: the K-tiles of two segments
        return [("gate", m, k, f, 0), ("gate", m, k, f, 1), ("rows", m, n, f), ("dgate", m, n, f), ("rows", m, k, both), ("weights", m, k, f, n)]

    wide = [plans(tmp_path, ask(*s)) for s in FFN_WIDE_SIZES]
    assert all(p[0] == "wide" for s in wide for p in s)
    assert any(int(p[1]) > 256 for s in wide for p in s) and any(int(p[1]) < 256 for s in wide for p in s)
    assert any(int(s[5][2]) > 1 for s in wide)                    # weights' gradients in K splits
    tiled = [plans(tmp_path, ask(*s)) for s in FFN_SIZES + FFN_SPLIT_SIZES if s[0] > 64]
    assert all(p[0] == "small" for s in tiled for p in s)
    assert all(any(int(s[i][2]) > 1 for s in tiled) and any(int(s[i][2]) == 1 for s in tiled) for i in (2, 4, 5))   # K splits of down, dx, weights
    long = plans(tmp_path, ask(4100, 4160, 131080, 200))
    assert long[4][0] == "wide" and long[5][0] == "wide" and 4160 % 192 in range(1, 129) and 4160 * 131080 > 2 ** 29
