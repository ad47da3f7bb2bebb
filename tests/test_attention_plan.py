"""How attention work is dealt out to CTAs (gv_attention_plan.h), played through on the host."""
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    out = str(tmp_path_factory.mktemp("plan") / "probe")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", out, os.path.join(HERE, "attention_plan_probe.cpp")], check=True)
    return out


def _run(probe, cases):
    text = "\n".join(f"{w} {step} {heads} {parts} {least} {len(seqs)} " + " ".join(f"{n} {length}" for n, length in seqs)
                     for w, step, heads, parts, least, seqs in cases)
    done = subprocess.run([probe], input=text, capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.strip() == f"ok {len(cases)}", done.stdout


def test_edges(probe):
    cases = []
    for window in (0, 1, 127, 128, 129, 1000):
        for step in (1, 16, 18, 25, 42, 64, 128, 256):
            cases.append((window, step, 3, 148, 4, [(1, 1), (1, 0), (0, 5), (5, 3), (700, 600), (300, 0), (129, 4000), (1, 128), (1, 129)]))
            cases.append((window, step, 1, 148, 1, [(0, 0), (2000, 2000), (0, 9)]))
            cases.append((window, step, 1, 7, 4, [(0, 0)]))
    _run(probe, cases)


def test_drawn(probe):
    rng = random.Random(5)
    cases = []
    for _ in range(600):
        seqs = [(rng.choice([0, 1, 1, 5, rng.randint(1, 900)]), rng.choice([0, 1, rng.randint(0, 300), rng.randint(0, 9000)]))
                for _ in range(rng.randint(1, 12))]
        cases.append((rng.choice([0, 0, 1024, rng.randint(1, 1500)]), rng.choice([1, 16, 32, 64, 128, 256, rng.randint(1, 256)]),
                      rng.randint(1, 16), rng.choice([1, 2, 148, 160]), rng.randint(1, 6), seqs))
    _run(probe, cases)
