"""The host rules of vvh_linear_q4 (linear_q4_plan and launch_linear_q4 of q4_kernels.hip) for a device of 256 CUs, so that
tests can say which way a shape takes.  They hold for the rules as they stand: a test that names a way asserts it here."""
from types import SimpleNamespace

CUS, STEP, TILE, LDS = 256, 256, 16 * 144 + 16 * 12 * 4, 160 * 1024


def up(a, b):
    return -(-a // b)


def lds_bytes(rows, seg, waves, f32):
    return (2 if f32 else 1) * rows * (seg * STEP + 8) * 2 + (seg * 16 * 4 if f32 else 0) + waves * TILE


def plan(M, N, K, f32):
    """kernel "rows" (x a step at a time) or "whole" (x staged whole); splits of k, floats of workspace; whole: waves a block,
    waves a tile (ks), groups of channels a block takes in turn (turns)."""
    tiles, steps, passes, rows = up(N, 16), up(K, STEP), up(M, 16), min(M, 16)
    groups, n16, n32 = up(N, 128), up(M, 16), up(M, 32)

    def stepwise(most, parts):
        n = up(M, most)
        seg = up(steps, parts)
        splits = up(steps, seg)
        return SimpleNamespace(kernel="rows", rows=up(M, n), seg=seg, splits=splits, ws=splits * M * N if splits > 1 else 0, turns=1)

    parts = min(up(CUS * 5 // 8, groups * n16), 12, steps)
    if M > (8 if f32 else 4) and groups * n16 >= CUS // 2:
        if parts > 1 and steps >= 12:
            return stepwise(16, parts)
        c16, c32 = up(groups * n16, CUS), up(groups * n32, CUS)
        return stepwise(32 if not f32 and 7 * c32 < 5 * c16 else 16, 1)
    p = SimpleNamespace(kernel="whole", splits=1, ks=1, waves=8, seg=max(2, steps))
    while lds_bytes(rows, p.seg, 8, f32) > (96 * 1024 if f32 and rows > 4 else LDS):
        p.splits += 1
        p.seg = max(2, up(steps, p.splits))
    if M > 4 and p.splits > 1:
        return stepwise(16, parts)
    while p.ks < 8 and p.ks < p.seg and tiles * passes * p.splits * p.ks < (4 if rows > 4 else 8) * CUS:
        p.ks *= 2
    p.waves = 8 if rows > 4 else max(4, p.ks)
    p.splits = up(steps, p.seg)
    p.ws = p.splits * M * N if p.splits > 1 else 0
    tpb = p.waves // p.ks
    p.groups = up(tiles, tpb)
    fit = max(1, min(LDS // lds_bytes(rows, p.seg, p.waves, f32), 32 // p.waves))
    worth, full = up(rows * (4 if f32 else 2), tpb), p.groups * passes * p.splits // (fit * CUS)
    p.turns = max(1, min(worth, full))
    p.slots = up(p.groups, p.turns)
    return p
