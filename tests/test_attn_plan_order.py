"""The plan of attention_paged's launches with sequences of long items first
(csrc/attn_plan.h, find_item<true>), run on the CPU lane by lane: every tile and split
once, in the parts of the plain order, and the items' lengths falling by sequence."""

import random
import subprocess
from pathlib import Path

import pytest

from test_attn_plan import BATCHES, _check

ROOT = Path(__file__).resolve().parents[1]
BM, BN, LONG = 128, 64, 24


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    path = tmp_path_factory.mktemp("plan")
    source = (ROOT / "tests" / "native" / "plan_lanes.cpp").read_text()
    ordered = source.replace("= find_item(", "= find_item<true>(").replace(
        "  args.Lmax =", "  args.longest = long_first(L);\n  args.Lmax =")
    assert ordered.count("find_item<true>(") == ordered.count("long_first(L)") == 1
    for name, text in (("plain", source), ("ordered", ordered)):
        (path / f"{name}.cpp").write_text(text)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas",
                        "-Wno-unused-function", "-ffp-contract=off", "-I",
                        str(ROOT / "mlir-toy_amd" / "csrc"), "-o", str(path / name),
                        str(path / f"{name}.cpp")], check=True)

    def form(name):
        def run(tokens, Hq, Hk, D, seq_kv, cu, lens, asked):
            text = [tokens, len(lens), Hq, Hk, D, seq_kv, 0 if cu is None else 1]
            text += ([] if cu is None else cu) + lens + [len(asked)] + list(asked)
            r = subprocess.run([path / name], input=" ".join(map(str, text)),
                               capture_output=True, text=True, check=True, timeout=100)
            room, *found = r.stdout.splitlines()
            return [int(x) for x in room.split()], [
                None if x == "-" else tuple(map(int, x.split())) for x in found]
        return run

    return form("plain"), form("ordered")


def _items(run, batch, Hq, Hk, D, seq_kv):
    cu = [sum(n for n, _ in batch[:b]) for b in range(len(batch) + 1)]
    lens = [n for _, n in batch]
    (items, *_), _ = run(cu[-1], Hq, Hk, D, seq_kv, cu, lens, [])
    return [x for x in run(cu[-1], Hq, Hk, D, seq_kv, cu, lens, range(items))[1] if x]


@pytest.mark.parametrize("batch,Hq,Hk,D,seq_kv,cut", BATCHES, ids=lambda x: str(x)[:24])
def test_items(built, batch, Hq, Hk, D, seq_kv, cut):
    assert (_check(built[1], batch, Hq, Hk, D, seq_kv) > 0) == cut
    assert sorted(_items(built[0], batch, Hq, Hk, D, seq_kv)) == sorted(
        _items(built[1], batch, Hq, Hk, D, seq_kv))


@pytest.mark.parametrize("batch,Hq,Hk,chain", [
    # (new, length): the shortest first, ties, sequences with nothing new between; the
    # last one's chain is short, though some of its items are not
    ([(422, 2409), (585, 4842), (277, 4300), (231, 5231)], 32, 8, True),
    ([(300, 4000), (0, 9000), (300, 4000), (700, 4000), (0, 0), (90, 6000)], 32, 8, True),
    ([(400, 3000 + 100 * i) for i in range(16)], 16, 16, True),
    ([(900, 2000), (1, 30000), (5, 12000)], 32, 4, False),
], ids=lambda x: str(x)[:24])
def test_long_items_come_first(built, batch, Hq, Hk, chain):
    longest = max(n for _, n in batch)
    plain, ordered = (_items(run, batch, Hq, Hk, 128, longest) for run in built)
    assert sorted(plain) == sorted(ordered)
    each = {b: -(-(-(-length // BN)) // splits) for b, _, _, length, _, _, _, splits, _ in ordered}
    came, seen = ([each[x[0]] for x in items] for items in (plain, ordered))
    assert max(each.values()) >= LONG
    want = sorted(came, reverse=True) if chain else came
    assert seen == want
    assert (ordered == plain) == (came == want)  # ties as they came
    # a sequence's tiles stay together, from the last
    for b in each:
        at = [i for i, x in enumerate(ordered) if x[0] == b]
        assert at == list(range(at[0], at[0] + len(at)))
        tiles = [ordered[i][4] for i in at]
        assert tiles == sorted(tiles, reverse=True)


def test_more_sequences_and_shorter_chains_come_in_order(built):
    for batch, Hq, Hk in (([(200, 3000 + 10 * i) for i in range(17)], 16, 4),
                          ([(20, 600), (30, 900), (40, 1400)], 8, 2),
                          ([(1, 30000), (1, 40000)], 8, 2)):
        longest = max(n for _, n in batch)
        plain, ordered = (_items(run, batch, Hq, Hk, 128, longest) for run in built)
        assert plain == ordered


def test_items_of_random_batches(built):
    rng = random.Random(12)
    for _ in range(40):
        Hq, Hk = rng.choice(((32, 8), (8, 1), (28, 7), (16, 16)))
        longest = rng.choice((2000, 9000, 30000))
        batch = [(rng.choice((0, 1, rng.randrange(900))), rng.randrange(-3, longest))
                 for _ in range(rng.choice((2, 3, 8, 16)))]
        if not sum(n for n, _ in batch):
            batch[0] = (1, batch[0][1])
        _check(built[1], batch, Hq, Hk, 128, longest)
        assert sorted(_items(built[0], batch, Hq, Hk, 128, longest)) == sorted(
            _items(built[1], batch, Hq, Hk, 128, longest))
