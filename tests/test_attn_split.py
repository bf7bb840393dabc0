"""How an attention call is split among work-groups (csrc/qm_attn_plan.h): the device code compiled for the CPU, a wave's lanes taking turns
(tests/cpu_wave). Every row tile's keys are taken once, partial results have slots of their own, and a row's first slot is one that some work-group writes:
the kernel that joins the pieces reads there where the others lie."""
import os
import random
import subprocess

import pytest

from arcinfer_amd import build

HERE = os.path.dirname(os.path.abspath(__file__))
TARGET = 512


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("split") / "split")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fwrapv", "-I", os.path.join(HERE, "cpu_wave"), "-I", build.CSRC, "-x", "c++",
                    os.path.join(HERE, "split_on_cpu.cpp"), "-o", exe], check=True)

    def run(RT, HK, G, T, start, lens, W, target=0, tail=0):
        B = len(lens)
        items = (T * G // RT + B if start else B * -(-G // RT)) * HK
        units = items + target + tail
        text = " ".join(map(str, [RT, HK, G, B, T, int(start is not None), W, 4, target, tail, units, 0, 1, *(start or []), *lens]))
        out = subprocess.run([exe], input=text, check=True, capture_output=True, text=True).stdout.split("\n")
        keys = ("unit", "b", "h", "rt", "c", "rts", "blocks", "more", "parts", "slot")
        return items, [dict(zip(keys, map(int, line.split()))) for line in out if line and line != "-1"]
    return run


def first_slot(RT, G, start, b, rt):
    return start[b] * G // RT + b + rt if start else b * -(-G // RT) + rt


def blocks_of(RT, G, rows, n, rt, W):
    """Blocks of 128 keys that the last row of a tile sees."""
    last = min((rt + 1) * RT, rows * G) - 1
    return (min(max(n - rows + last // G + 1, 0), 16 * W) + 127) // 128


@pytest.mark.parametrize("kind", ["whole", "cut", "tail", "many"])
@pytest.mark.parametrize("seed", range(6))
def test_batches(split, kind, seed):
    r = random.Random(seed)
    RT, HK, G = r.choice((64, 128) if kind == "tail" else (16, 32, 64, 128)), r.choice((1, 2, 3, 8)), r.choice((1, 2, 5, 8))
    B, most, listed = r.choice((1, 3, 70, 200)), r.choice((1, 3, 90)), seed % 3 > 0
    if kind == "tail":
        B, most, listed, HK = r.choice((1, 3, 20)), 300, True, 8
    if kind == "many":
        RT, B, most = 16, 270, 3
    rows = [r.randint(0, most) if listed else 1 for _ in range(B)]
    rows[-1] = max(1, rows[-1])
    W = 2000
    lens = [min(16 * W + 5, n + int(2 ** r.uniform(0, 15))) for n in rows]
    start = [sum(rows[:b]) for b in range(B + 1)] if listed else None
    T = sum(rows) + (3 if listed else 0)
    target = r.choice((1, 7, TARGET)) if kind == "cut" else 0
    tail = TARGET if kind == "tail" else 0
    items, done = split(RT, HK, G, T, start, lens, W, target, tail)
    taken, slots = {}, set()
    for i in done:
        n = -(-rows[i["b"]] * G // RT)
        assert 0 <= i["h"] < HK and i["rts"] == n and 0 <= i["rt"] < n
        all_blocks, per = blocks_of(RT, G, rows[i["b"]], lens[i["b"]], i["rt"], W), i["blocks"]
        if i["slot"] >= 0:
            assert i["slot"] < TARGET
            per = max(-(-all_blocks // i["parts"]), 4) if i["parts"] > 1 else 1 << 30
        if i["c"] and i["c"] * per >= all_blocks:
            continue  # (a piece that the tile's rows do not see: the work-group returns)
        keys = taken.setdefault((i["b"], i["h"], i["rt"]), [])
        keys += range(i["c"] * per, min((i["c"] + 1) * per, all_blocks))
        if target:
            others = items // HK + i["more"] + i["rt"]
            at = others + (i["c"] - 1) * i["rts"] if i["c"] else first_slot(RT, G, start, i["b"], i["rt"])
            assert at * HK + i["h"] < items + target and (at, i["h"]) not in slots
            slots.add((at, i["h"]))
    for b in range(B):
        for h in range(HK):
            for rt in range(-(-rows[b] * G // RT)):
                assert sorted(taken[b, h, rt]) == list(range(blocks_of(RT, G, rows[b], lens[b], rt, W)))
                assert not target or (first_slot(RT, G, start, b, rt), h) in slots
    assert len(taken) == HK * sum(-(-n * G // RT) for n in rows)


@pytest.mark.parametrize("kind", ["whole", "cut", "tail", "many"])
def test_lists_that_are_no_batch(split, kind):
    """Descending ones: nothing outside the call's rows, heads and slots. Some rows' first slots are written by nobody, which is why the join takes no word of
    a slot unseen."""
    unwritten = 0
    for start in ([0, 90] * 8, [90, 0, 90, 0, 0], [-5, 90, 20, 2 ** 31 - 1, -2 ** 31, 7]):
        RT, HK, G, T, B = 64 if kind == "tail" else 16, 2, 4, 90, len(start) - 1
        if kind == "many":
            start = start * 60
            B = len(start) - 1
        lens, target, tail = [3000] * B, TARGET - 60 if kind == "cut" else 0, TARGET if kind == "tail" else 0
        items, done = split(RT, HK, G, T, start, lens, 200, target, tail)
        at = [min(max(s, 0), T) for s in start]
        slots = set()
        for i in done:
            rows = max(at[i["b"] + 1] - at[i["b"]], 0)
            assert 0 <= i["b"] < B and 0 <= i["h"] < HK and 0 <= i["rt"] < -(-rows * G // RT) and -1 <= i["slot"] < TARGET and i["c"] >= 0
            if i["c"] == 0:
                slots.add(first_slot(RT, G, at, i["b"], i["rt"]))
        for t in range(T):  # (the sequence that the join finds for row t)
            lo, hi = 0, B
            while lo < hi:
                mid = (lo + hi + 1) // 2
                lo, hi = (mid, hi) if start[mid] <= t else (lo, mid - 1)
            if lo < B and at[lo] <= t < at[lo + 1]:
                unwritten += first_slot(RT, G, at, lo, (t - at[lo]) * G // RT) not in slots
    assert kind != "cut" or unwritten > 0
