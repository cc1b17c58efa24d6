"""How attention over many rows is divided over workgroups (csrc/dm_attend_walk.h), gone over
on the host by attend_walk.cpp: every step of every unit is done once, units that lie in several
workgroups are counted alike by all of them, and no walk leaves the line or runs on."""
import os
import random
import subprocess

import pytest

from conftest import PKG

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    exe = tmp_path_factory.mktemp("walk") / "attend_walk"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-ftrapv", "-I",
                    os.path.join(PKG, "csrc"), os.path.join(HERE, "attend_walk.cpp"), "-o", str(exe)],
                   check=True)

    def run(batches):
        text = "\n".join(f"{rep} {heads} {max(rep, 64)} {grid} {len(seqs)} "
                         + " ".join(f"{n} {past}" for n, past in seqs)
                         for rep, heads, grid, seqs in batches)
        r = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stdout
        assert r.stdout.strip() == f"{len(batches)} batches"
    return run


def test_ratios_that_are_no_power_of_two(walk):
    """Prompts whose places on a line of fractions would differ from lane to lane."""
    walk([(5, 8, 512, [(700, 0), (700, 1000), (1000, 0)]),
          (7, 4, 512, [(256, 1000), (300, 500), (300, 100)]),
          (6, 1, 512, [(339, 1769), (530, 578), (741, 0)]),
          (3, 4, 512, [(148, 0), (306, 1288), (316, 0)]),
          (6, 4, 512, [(654, 381), (868, 99), (668, 1820), (1, 0), (897, 0), (1, 0)])])


def _batch(r, num, most, rep=None):
    seqs = []
    for _ in range(num):
        kind = r.random()
        # prompts, single tokens, skipped and empty sequences
        n = r.randint(2, most) if kind < 0.6 else 1 if kind < 0.85 else 0
        seqs.append((n, r.choice([0, 0, r.randint(1, 200), r.randint(1, 5000)])))
    return (rep or r.randint(1, 17), r.choice([1, 2, 3, 4, 5, 8]), r.choice([256, 512]), seqs)


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(walk, seed):
    r = random.Random(seed)
    walk([_batch(r, r.randint(1, 12), 1000) for _ in range(400)]
         + [_batch(r, r.randint(13, 600), 90) for _ in range(25)]
         + [_batch(r, r.randint(250, 260), 40) for _ in range(5)])


def test_small_grids_and_large_ratios(walk):
    r = random.Random("grids")
    walk([(rep, heads, grid, [(n, past), (1, 7), (n + 1, 0)])
          for rep in (1, 16, 24, 66, 127, 128, 129, 4096) for heads in (1, 3)
          for grid in (1, 2, 7, 512) for n, past in ((2, 0), (r.randint(65, 300), 70), (130, 40000))])


def test_one_row_more_than_few(walk):
    """Sequences at the limit from which there are units, alone and beside each other."""
    walk([(rep, 2, 512, [(n, past)] * k) for rep in (1, 2, 3, 64, 65) for past in (0, 1, 63, 64)
          for n in (max(rep, 64) // rep, max(rep, 64) // rep + 1) for k in (1, 2, 5)])


def test_the_longest_lines(walk):
    """Lengths stay within 64 bits for contexts of 2^30 tokens (a whole unit is some 2^36 long)."""
    far = (1 << 30) - 5000
    walk([(1, 1, 512, [(2000, far)] * 40), (3, 8, 512, [(4000, far), (1, far), (700, far)]),
          (4096, 1, 512, [(60, far)]), (129, 16, 256, [(300, far), (0, 0), (77, far)]),
          (1, 1, 512, [(1 << 22, 0)]), (16, 2, 512, [(1 << 18, 1 << 20)])])
