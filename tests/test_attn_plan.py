"""The plan of attention_paged's launches (csrc/attn_plan.h), run on the CPU lane by
lane: the items of a launch cover every tile and split once, states stay within the
room that the workspace has for them, and sequences that overlap are not cut."""

import random
import subprocess
from pathlib import Path

import pytest

from test_gpu_attention_paged_cuts import CUTS

ROOT = Path(__file__).resolve().parents[1]
BM = 128


@pytest.fixture(scope="module")
def lanes(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "plan_lanes"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas",
                    "-Wno-unused-function", "-ffp-contract=off", "-I",
                    str(ROOT / "mlir-toy_amd" / "csrc"), "-o", str(exe),
                    str(ROOT / "tests" / "native" / "plan_lanes.cpp")], check=True)

    def run(tokens, Hq, Hk, D, seq_kv, cu, lens, asked):
        text = [tokens, len(lens), Hq, Hk, D, seq_kv, 0 if cu is None else 1]
        text += [] if cu is None else cu
        text += lens + [len(asked)] + list(asked)
        r = subprocess.run([exe], input=" ".join(map(str, text)), capture_output=True, text=True,
                           check=True, timeout=100)
        room, *found = r.stdout.splitlines()
        return [int(x) for x in room.split()], [None if x == "-" else tuple(map(int, x.split()))
                                                for x in found]

    return run


def _check(lanes, batch, Hq, Hk, D, seq_kv):
    """Items of a launch of sequences [(new, length)], each once, states apart."""
    cu = [sum(n for n, _ in batch[:b]) for b in range(len(batch) + 1)]
    lens = [n for _, n in batch]
    (items, _, parts, *_), _ = lanes(cu[-1], Hq, Hk, D, seq_kv, cu, lens, [])
    _, found = lanes(cu[-1], Hq, Hk, D, seq_kv, cu, lens, range(items))
    want = {(b, t) for b, (n, _) in enumerate(batch) for t in range(-(-n * (Hq // Hk) // BM))}
    got, states, cut = {}, set(), 0
    for it in filter(None, found):
        b, n, row0, length, tile, tiles, split, splits, part = it
        assert (n, row0, length) == (batch[b][0], cu[b], min(max(batch[b][1], 0), seq_kv))
        assert 0 <= split < splits
        assert (b, tile, split) not in got
        got[b, tile, split] = splits
        if splits > 1:
            cut += 1
            assert 0 <= part and part + split < parts, "a state without room"
            assert part + split not in states
            states.add(part + split)
    assert {(b, t) for b, t, _ in got} == want
    assert all(sum(1 for s in range(n) if (b, t, s) in got) == n for (b, t, _), n in got.items())
    return cut


BATCHES = [
    # (batch, Hq, Hk, D, longest, whether keys are cut)
    ([(1, 1)], 8, 2, 128, 1, False),
    ([(1, 32768)], 32, 8, 128, 32768, True),
    ([(1, 3000)], 32, 8, 128, 3000, True),
    ([(4, 8000)] * 16, 32, 8, 128, 8000, True),
    ([(1, 8000)] * 32, 32, 8, 128, 8000, True),
    ([(4096, 4096)] * 4, 32, 8, 128, 4096, False),
    ([(1000, 31000)], 32, 8, 128, 31000, True),
    ([(500, 8000)] + [(1, 8000)] * 7, 32, 8, 128, 8000, True),
    ([(130, 1500), (1, 1), (0, 300), (0, 0), (77, 900)], 16, 4, 64, 1500, True),
    ([(0, 40)] * 700 + [(2, 1500)] + [(0, 0)] * 100 + [(1, 700)], 8, 2, 64, 1500, True),
    ([(1, 600), (3, 530)], 513, 513, 64, 600, False),
    ([(3, -5), (140, 100), (2, 7)], 8, 2, 64, 900, False),
    ([(2, 9000)] * 3, 8, 1, 64, 640, True),  # longer than the bound: cut down to it
]


@pytest.mark.parametrize("batch,Hq,Hk,D,seq_kv,cut", BATCHES, ids=lambda x: str(x)[:24])
def test_items(lanes, batch, Hq, Hk, D, seq_kv, cut):
    assert (_check(lanes, batch, Hq, Hk, D, seq_kv) > 0) == cut


@pytest.mark.parametrize("batch,Hq,Hk,D,page,qt,kt,cut,groups", CUTS, ids=lambda x: str(x)[:24])
def test_what_the_gpu_tests_mean_to_cut(lanes, batch, Hq, Hk, D, page, qt, kt, cut, groups):
    longest = max(n for _, n in batch)
    assert (_check(lanes, batch, Hq, Hk, D, longest) > 0) == cut
    (_, _, parts, _, by), _ = lanes(sum(n for n, _ in batch), Hq, Hk, D, longest, None,
                                    [n for _, n in batch], [])
    assert parts > 0 and by == groups


def test_items_of_random_batches(lanes):
    rng = random.Random(11)
    for _ in range(60):
        Hq, Hk = rng.choice(((32, 8), (8, 1), (28, 7), (4, 4), (12, 12), (16, 1)))
        B = rng.choice((1, 2, 5, 30, 63, 64, 65, 90))
        longest = rng.choice((500, 900, 3000, 20000))
        batch = []
        for _ in range(B):
            n = rng.choice((0, 1, 1, 2, 5, rng.randrange(300)))
            batch.append((n, rng.randrange(-3, longest)))
        if not sum(n for n, _ in batch):
            batch[0] = (1, batch[0][1])
        _check(lanes, batch, Hq, Hk, rng.choice((64, 128)), longest)


@pytest.mark.parametrize("B,tokens,Hq,Hk,length", [
    (40, 64, 8, 2, 900), (2000, 64, 8, 1, 6000), (1 << 16, 1 << 23, 1, 1, 6000),
    (1 << 16, 1 << 19, 16, 1, 0)], ids=str)
def test_states_of_sequences_that_overlap_stay_within_the_room(lanes, B, tokens, Hq, Hk, length):
    """cu_seqlens that run back name rows again and again. Whatever is cut, a state lies
    within the room: tiles times splits of what is cut is at most tiles times blocks over
    the chain, and the chain is at least the launch's blocks over 512 work-groups, summed
    in 64 bits."""
    cu = [0, tokens] * (B // 2) + [tokens]
    lens = [length] * B
    (items, _, parts, *_), _ = lanes(tokens, Hq, Hk, 64, 6000, cu, lens, [])
    assert parts > 0, "keys could be cut"
    asked = sorted({0, 1, 2, parts - 1, parts, parts + 1, items // 2, items - 2, items - 1})
    _, found = lanes(tokens, Hq, Hk, 64, 6000, cu, lens, [i for i in asked if 0 <= i < items])
    for b, n, row0, length, tile, tiles, split, splits, part in filter(None, found):
        assert splits == 1 or 0 <= part + split < parts


@pytest.mark.parametrize("B,rows,group", [
    (200, 1 << 14, 1),
    # every other sequence names all rows but the first: 2^31 tiles in all, 2^38 rows
    (1 << 16, 1 << 23, 1), (1 << 16, 1 << 23, 16),
    (1 << 16, 3 << 21, 1),  # 3 2^29 tiles
], ids=str)
def test_more_tiles_than_the_launch_has_items_for_are_not_cut(lanes, B, rows, group):
    """The first sequence, one token over many keys, would be cut but for the others."""
    tokens = rows // group + 1
    cu = [0] + [1, tokens] * (B // 2)
    lens = [100000] + [0] * (B - 1)
    (items, _, parts, *_), found = lanes(tokens, group, 1, 64, 100000, cu, lens, [0, 1, 2])
    assert parts > 0, "keys could be cut"
    assert [it[7] for it in found] == [1, 1, 1]
    # and it is, by itself
    assert lanes(1, group, 1, 64, 100000, [0, 1], lens[:1], [0])[1][0][7] > 1
