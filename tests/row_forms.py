"""Which kernel the row attention takes for a call, restated from the rules in attend_rows.hip and kernels.hip
(rows_decode_ok, rows_mfma_ok, long_plan, launch_tile, launch_mfma, launch_decode), and the calls that the GPU tests
make so that each of them runs. Not what the kernels compute: attention_ref.py has that."""

ROWS, TABLE_MOST = 16, 16384


def up(x, n):
    return -(-x // n)


def long_plan(b, t, h, hd, cap):
    """(row tiles, tiles of a group, key ranges, keys of a range)"""
    tiles = up(t, ROWS)
    wt = 4 if tiles >= 3 else tiles
    ng = max(1, min(1024 // (b * h * up(tiles, wt)), up(cap, 512)))
    ng = max(ng, up(cap, 65536))
    span = up(up(cap, ng), 256) * 256
    return tiles, wt, up(cap, span), span


def split_chunks(rh, cap):
    blocks = up(cap, 64)
    return up(cap, min(4096, 64 * up(blocks, max(1, min(up(4096, rh), blocks)))))


def mfma(b, t, h, hd, cap, table):
    tiles, panels = up(t, ROWS), b * h + 7
    if hd % 16 or table > TABLE_MOST or panels * tiles >= 1 << 23:
        return False
    if cap <= 2048:
        return True
    _, wt, ng, _ = long_plan(b, t, h, hd, cap)
    return panels * up(tiles, wt) * ng * (up(hd, 64) if hd > 128 else 1) < 1 << 24 and \
        panels * tiles * ROWS * (hd // 4) < (1 << 32) - 256


def one_launch(rh, hd, cap):
    return hd in (16, 32, 64, 128) and cap <= 1024 and (hd != 128 or cap <= 128 or rh <= 1024)


def decode(b, t, h, hd, cap, table, mass):
    rh = b * h
    return mass and t == 1 and hd in (16, 32, 64, 128, 256) and rh < 1 << 22 and \
        (one_launch(rh, hd, cap) or not mfma(b, t, h, hd, cap, table) or (cap > 2048 and rh >= 512))


def form(b, t, h, hd, cap, score_s, mass, table=8192):
    """The kernels of a call whose arrays are aligned to 16 bytes (score_m past -2^31)."""
    if decode(b, t, h, hd, cap, table, mass):
        noclamp = score_s >= 13
        if not one_launch(b * h, hd, cap):
            return "split", hd, noclamp
        if cap > {128: 128, 64: 256}.get(hd, 512):
            return "workgroup", hd, noclamp
        kb = up(cap, 64)
        return "wave", hd, kb if kb <= 4 else 8, noclamp
    if not mfma(b, t, h, hd, cap, table):
        return ("rows",)
    qc, hi = 1 if hd <= 64 else 2 if hd <= 128 else 4, 32 <= score_s <= 60
    tiles, wt, ng, _ = long_plan(b, t, h, hd, cap)
    if cap > 2048 or (cap > 1024 and tiles >= 3 and ng == 1):
        return "walks", qc, wt, hi, ng == 1
    if cap <= 512:
        return "tile", qc, 1 if cap <= 256 else 2, 4, hi
    if cap <= 1024:
        return ("tile", qc, 4, 4, hi) if qc > 1 and b * h * tiles > 256 else ("tile", qc, 2, 8, hi)
    return "tile", qc, 4, 8, hi


def workspace(b, t, h, hd, cap, mass, table=8192):
    """The bytes that the call's form needs, 0 where none."""
    al = lambda x: up(x, 256) * 256  # noqa: E731
    kind = form(b, t, h, hd, cap, 36, mass, table)
    if kind[0] == "split":
        rh, chunks = b * h, split_chunks(b * h, cap)
        return al(rh * cap * 4) + 2 * al(rh * chunks * 8) + al(rh * chunks * hd * 8)
    if kind[0] != "walks" or kind[4]:
        return 0
    tiles, _, ng, _ = long_plan(b, t, h, hd, cap)
    rows = b * h * tiles * ROWS
    return 2 * al(rows * ng * 8) + rows * ng * hd * 8


# Every form of the fast kernels.
FORMS = [("tile", qc, nb, nw, hi) for qc in (1, 2, 4) for nb, nw in ((1, 4), (2, 4), (4, 4), (2, 8), (4, 8))
         for hi in (True, False) if (qc, nb, nw) != (1, 4, 4)]
FORMS += [("walks", qc, wt, hi, alone) for qc in (1, 2, 4) for wt in (1, 2, 4) for hi in (True, False)
          for alone in (True, False)]
DECODE_FORMS = [("wave", hd, kb, n) for hd, kbs in ((16, (1, 2, 3, 4, 8)), (32, (1, 2, 3, 4, 8)), (64, (1, 2, 3, 4)), (128, (1, 2)))
                for kb in kbs for n in (True, False)]
DECODE_FORMS += [("workgroup", hd, n) for hd in (16, 32, 64, 128) for n in (True, False)]
DECODE_FORMS += [("split", hd, n) for hd in (16, 32, 64, 128, 256) for n in (True, False)]

# Rules of one scale (about 0.02 a dot) by their score shift: in and out of 32 ..= 60, and where scores are clamped.
SCORES = {36: 1_400_000_000, 22: 85_449, 8: 5}

# Calls (b, t, h, hd, cap) that are run as a tree and as a causal chunk, with the shifts 36 and 22 or 8.
SHAPES = [(3, t, 2, hd, cap) for hd in (64, 128, 256) for t, cap in ((20, 200), (5, 400), (40, 900), (20, 1900))]
SHAPES += [(130, 20, 1, hd, 900) for hd in (128, 256)]                                 # more than 256 workgroups
SHAPES += [(3, t, 2, hd, 2600) for hd in (64, 128, 256) for t in (5, 20, 40)]          # ranges of keys
SHAPES += [(520, t, 1, hd, 2052) for hd in (64, 128, 256) for t in (5, 20)]            # a workgroup a cache
SHAPES += [(520, 40, 1, hd, 1100) for hd in (64, 128, 256)] + [(520, 70, 1, 64, 2052)]
SHAPES += [(2, 33, 1, hd, 5000) for hd in (80, 192)]                                   # part of a channel group, a wave without rows

# Calls (b, h, hd, cap) of one row with weights.
ONE_ROW = [(5, 2, hd, cap) for hd in (16, 32, 64, 128) for cap in (60, 120, 180, 250, 500, 900)]
ONE_ROW += [(520, 1, hd, 2100) for hd in (16, 32, 64, 128, 256)]
