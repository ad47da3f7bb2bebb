"""The shares of attention work that every CTA takes, and what the join finds of them (attn_walk in gv_attention_plan.h), played through on the host."""
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def compile_probe(folder, header=None):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    source = os.path.join(HERE, "attention_walk_probe.cpp")
    if header is not None:  # another text of the plan
        with open(source) as f:
            text = f.read().replace("../gevva_b200/csrc/gv_attention_plan.h", "plan.h")
        source = os.path.join(folder, "probe.cpp")
        for name, content in (("probe.cpp", text), ("plan.h", header)):
            with open(os.path.join(folder, name), "w") as f:
                f.write(content)
    out = os.path.join(folder, "probe")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", out, source], check=True)
    return out


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    return compile_probe(str(tmp_path_factory.mktemp("walk")))


def run(probe, cases):
    text = "\n".join(f"{w} {step} {heads} {parts} {least} {len(seqs)} " + " ".join(f"{n} {length}" for n, length in seqs)
                     for w, step, heads, parts, least, seqs in cases)
    return subprocess.run([probe], input=text, capture_output=True, text=True, timeout=300)


def check(probe, cases):
    done = run(probe, cases)
    assert done.returncode == 0 and done.stdout.strip() == f"ok {len(cases)}", done.stdout


def edges():
    for window in (0, 1, 127, 128, 129, 1000):
        for step in (1, 16, 18, 25, 42, 64, 128, 256):
            for parts in (1, 7, 148):
                yield window, step, 3, parts, 1, [(1, 1), (1, 0), (0, 5), (5, 3), (700, 600), (300, 0), (129, 4000), (1, 128), (1, 129)]
                yield window, step, 1, parts, 1, [(0, 0), (2000, 2000), (0, 9)]
                # runs inside one sequence, shorter and longer than an item, that begin and end inside items
                yield window, step, 2, parts, 1, [(4096, 4096 + 37)]
                yield window, step, 1, parts, 1, [(512, 32000)]
                yield window, step, 16, parts, 1, [(1, 20000)]


def drawn():
    rng = random.Random(8)
    for _ in range(500):
        seqs = [(rng.choice([0, 1, 1, 5, rng.randint(1, 900)]), rng.choice([0, 1, rng.randint(0, 300), rng.randint(0, 9000)]))
                for _ in range(rng.randint(1, 70))]
        if not any(n for n, _ in seqs):
            seqs[0] = (1, 1)
        yield (rng.choice([0, 0, 1024, rng.randint(1, 1500)]), rng.choice([1, 16, 32, 64, 128, 256, rng.randint(1, 256)]), rng.randint(1, 16),
               rng.choice([1, 2, 148, 160, 1100]), rng.randint(1, 6), seqs)


def test_edges(probe):
    check(probe, list(edges()))


def test_drawn(probe):
    check(probe, list(drawn()))


def test_work_past_the_divisions_in_32_bits(probe):
    """From 2^22 key tiles on, and with more than 1023 parts, on both sides of either line."""
    million = 1 << 20
    check(probe, [(0, 128, 8, 148, 1, [(1, million)] * 64), (0, 128, 8, 148, 1, [(1, million)] * 64 + [(1, 1)]),
                  (0, 128, 1, 148, 1, [(1, 128 * ((1 << 22) - 1))]), (0, 128, 1, 148, 1, [(1, 128 << 22)]), (0, 128, 1, 1023, 1, [(1, 128 << 22)]),
                  (0, 128, 3, 1024, 1, [(7, 10000000), (300, 9999999)]), (0, 16, 2, 148, 1, [(4096, 40 * million)]),
                  (5000, 64, 8, 148, 1, [(100000, 101234)] * 5)])


def test_lengths_that_change_while_a_call_runs(probe):
    """As when another stream writes them: the results are then wrong, but every CTA ends and stays within its workspace."""
    done = subprocess.run([probe, "change"], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout


@pytest.mark.parametrize("line,wrong", [
    ("share.slot = share.take == tiles ? -1 : 2 * part + (share.skip == 0 ? 1 : 0);", "share.slot = share.take == tiles ? -1 : 2 * part;"),
    ("share.behind = upto - part;", "share.behind = upto - part - 1;"),
    ("share.behind = upto - part;", "share.behind = upto - part + 1;"),
    ("          offset = first_offset;", "          offset = 0;"),
    ("stop = end - (target + 1 - before);", "stop = end - (target - before);"),
    ("if (last >= 0) at = end;", "")])
def test_a_plan_that_is_wrong_does_not_pass(tmp_path, line, wrong):
    """The check itself: with one line of the plan another, it fails."""
    with open(os.path.join(HERE, "..", "gevva_b200", "csrc", "gv_attention_plan.h")) as f:
        text = f.read()
    assert text.count(line) == 1
    done = run(compile_probe(str(tmp_path), text.replace(line, wrong)), list(edges()))
    assert done.returncode == 1, done.stdout
